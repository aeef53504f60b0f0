"""Argument checks that the operators on rows over a vocabulary share
(``ops.embedding``, ``ops.logprobs``, ``ops.distill``)."""
from __future__ import annotations

import contextlib
import sys
from typing import Optional

import torch
from torch.autograd import forward_ad

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # vocab_common.hpp kF32, kBF16, kF16
_NOTHING = contextlib.nullcontext()
_tracing = torch._C._get_tracing_state
_modes = torch._C._len_torch_dispatch_stack
_functions = torch._C._len_torch_function_stack
_RECORDING = (torch._C._TorchDispatchModeKey.FAKE, torch._C._TorchDispatchModeKey.FUNCTIONAL)


def _traced() -> bool:
    """Whether torch.jit.trace, make_fx or a fake mode records the calls made
    here (other modes, such as a default device or a counter of operations, do not)."""
    if _tracing() is not None:
        return True
    proxy = sys.modules.get("torch.fx.experimental.proxy_tensor")   # (its import takes long, and make_fx is in it)
    if proxy is not None and proxy.get_proxy_mode() is not None:
        return True
    return _modes() > 0 and any(torch._C._get_dispatch_mode(k) is not None for k in _RECORDING)


def no_grad_of(grad_name: str, *tensors) -> None:
    """These operators are not recorded by autograd; their gradients are
    functions of their own.  A tensor that autograd follows, backwards or
    forwards, is refused rather than dropped out of its graph without a word,
    and so is a call that a tracer records: it would see the output's
    allocation and no kernel."""
    if (_tracing() is not None or _modes() or _functions()) and _traced():
        raise ValueError("a tracer does not see what this operator computes: call it outside of torch.jit.trace, "
                         "make_fx and fake tensor modes")
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"autograd does not follow this operator: call it under torch.no_grad() or on a detached "
                             f"tensor, and {grad_name} for the gradient")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("forward-mode differentiation does not follow this operator: call it on the primal "
                                 "(torch.autograd.forward_ad.unpack_dual), without the tangent")


# (A view may hold the negatives of its values and a bit that says so, as the imaginary part of a
# conjugate does: resolve_neg() puts the values in memory.)

def contiguous(x: torch.Tensor) -> torch.Tensor:
    if x.is_neg():
        x = x.resolve_neg()
    return x if x.is_contiguous() else x.contiguous()


def matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as [rows, columns] of one of the three types with adjacent columns
    (copied if they are not adjacent; any row stride)."""
    if x.dim() != 2:
        raise ValueError(f"{what} must have 2 dimensions, got {tuple(x.shape)}")
    if x.dtype not in TYPES:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {x.dtype}")
    if x.is_neg():
        x = x.resolve_neg()
    if x.stride()[1] != 1 and x.shape[1] > 1:
        return x.contiguous()
    return x


def same_device(device: torch.device, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the other operands on {device}")


def on_cpu(x: torch.Tensor) -> bool:
    """True; operands that are neither on a GPU nor on the CPU are refused."""
    if not x.is_cpu:
        raise ValueError(f"operands must be on the CPU or a GPU, got {x.device}")
    return True


def token_ids(tokens: torch.Tensor) -> torch.Tensor:
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.is_neg():
        tokens = tokens.resolve_neg()
    return tokens if tokens.is_contiguous() else tokens.contiguous()


def per_row(x: Optional[torch.Tensor], n: int, what: str) -> Optional[torch.Tensor]:
    """A number for each row, fp32 (a broadcast one is laid out)."""
    if x is None:
        return None
    if x.dim() != 1 or x.shape[0] != n:
        raise ValueError(f"{what} must be [{n}], got {tuple(x.shape)}")
    if not x.is_floating_point():
        raise ValueError(f"{what} must be floating point, got {x.dtype}")
    if x.dtype != torch.float32:
        x = x.float()
    return contiguous(x)


def output(out: torch.Tensor, shape, dtype: torch.dtype, device: torch.device, what: str = "out") -> None:
    """A caller's output: the right shape, type and device, adjacent columns,
    rows that do not overlap each other."""
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(out.shape)}")
    if out.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {out.dtype}")
    same_device(device, **{what: out})
    if out.is_neg():
        raise ValueError(f"{what} must not have its negative bit set")
    if out.dim() == 2:
        n, d = out.shape
        if (d > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < d):
            raise ValueError(f"{what} must have adjacent columns and rows that do not overlap, got strides "
                             f"{out.stride()}")
    elif not out.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices with adjacent columns share an element."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    ea, eb = a.element_size(), b.element_size()
    la, lb = a.stride(0) * ea, b.stride(0) * eb
    wa, wb = a.shape[1] * ea, b.shape[1] * eb
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + (a.shape[0] - 1) * la + wa <= pb or pb + (b.shape[0] - 1) * lb + wb <= pa:
        return False
    if la == lb and la > 0 and a.shape[0] > 1 and b.shape[0] > 1:   # columns of the same rows
        off = (pb - pa) % la
        return not (off >= wa and off + wb <= la)
    return True


def apart(out: torch.Tensor, x: torch.Tensor, what: str, in_place: bool) -> None:
    """out does not share memory with x, unless it is x itself and that is allowed."""
    if overlaps(out, x):
        same = out.data_ptr() == x.data_ptr() and out.dtype == x.dtype and (out.shape[0] == 1 or
                                                                             out.stride(0) == x.stride(0))
        if not (in_place and same):
            raise ValueError(f"out overlaps {what}" + (f" without being {what} itself" if in_place else ""))


def inverse_temperature(temperature: float) -> float:
    t = float(temperature)
    if not 1e-30 < t < 1e30:
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return 1.0 / t


def on(device: torch.device):
    """Launches go to the current device: make it the operands'."""
    return _NOTHING if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)
