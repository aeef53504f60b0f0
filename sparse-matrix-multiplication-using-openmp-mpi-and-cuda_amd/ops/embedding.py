"""Embedding lookup with scaling and its gradient by sorted tokens.

The lookup is the product ``Y = scale * S W`` of the one-hot CSR matrix S of
the tokens (one row a token) with a dense table, the gradient the transposed
product ``dW = scale * S^T dY``.  Unlike :func:`ops.spmm.spmm` it needs no CSR
arrays, takes fp32, bf16 and fp16 and any width, and reads every row once.

* Token -1 is padding: its row of Y is zero and it adds nothing to dW.
* A token that the table does not have (below -1, or V and above) gives a row
  of NaN and adds nothing to dW: checking it on the host would wait for the GPU.
* Sums are held in fp32, over ascending positions in parts that the sizes
  determine, and rounded once: results are the same in every run.

gfx950 kernels: ``csrc/kernels/embedding.hip``; CPU tensors use the OpenMP
kernels of ``csrc/host/vocab_cpu.cpp``.  Nothing here waits for the GPU, so
both directions can be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from .. import _native
from .._native import c_vp, null
from . import rows as R

_native.register_hip("spmm_embedding", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, C.c_int, C.c_int64,
                     C.c_float, c_vp, C.c_int64, c_vp)
_native.register_hip("spmm_embedding_grad_ws", C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int64, C.c_int,
                     restype=C.c_int64)
_native.register_hip("spmm_embedding_grad", c_vp, C.c_int64, C.c_int, c_vp, C.c_int, C.c_int64, C.c_int64, C.c_int64,
                     C.c_float, c_vp, C.c_int64, C.c_int, C.c_int, c_vp, C.c_int64, c_vp)


def _scale(scale: float) -> float:
    s = float(scale)
    if not -3e38 <= s <= 3e38:
        raise ValueError(f"scale must be finite, got {scale}")
    return s


def embedding(W: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * W[tokens]``, [*tokens.shape, D], of W's type.

    W: [V, D] fp32, bf16 or fp16, rows at any stride; tokens: int32 or int64 of
    any shape.  ``out`` (that shape and type; rows may be strided where tokens
    has one dimension) is written instead of a new tensor."""
    R.no_grad_of("embedding_grad", W)
    W = R.matrix(W, "W")
    dev = W.device
    if tokens.device != dev:
        R.same_device(dev, tokens=tokens)
    gpu = W.is_cuda or not R.on_cpu(W)
    tok = R.token_ids(tokens)
    scale = _scale(scale)
    V, D = W.shape
    n = tok.numel()
    if out is None:
        out = torch.empty(*tokens.shape, D, dtype=W.dtype, device=dev)   # (a tuple costs 0.4 us more)
    else:
        R.no_grad_of("embedding_grad", out)
        R.output(out, (*tokens.shape, D), W.dtype, dev)
        R.apart(out if out.dim() == 2 else out.view(n, D), W, "W", in_place=False)
    if n == 0 or D == 0:
        return out
    y = out if out.dim() == 2 else out.view(n, D)
    at_w, at_tok, at_y = W.data_ptr() or null(W), tok.data_ptr() or null(tok), y.data_ptr() or null(y)
    if not gpu:
        w, t = W.float().contiguous(), tok.to(torch.int64)
        acc = torch.empty((n, D), dtype=torch.float32)
        _native.check(_native.host().spmm_cpu_embedding(n, V, D, _native.ptr(w), _native.ptr(t), scale,
                                                        _native.ptr(acc), 0), "cpu_embedding")
        y.copy_(acc)
        return out
    with R.on(dev):
        _native.check(_native.hip().spmm_embedding(at_w, W.stride(0), V, D, R.TYPES[W.dtype], at_tok,
                                                   tok.dtype == torch.int64, n, scale, at_y, y.stride(0),
                                                   R.stream(dev)), "embedding")
    return out


def embedding_grad(dY: torch.Tensor, tokens: torch.Tensor, V: int, scale: float = 1.0,
                   dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                   accumulate: bool = False) -> torch.Tensor:
    """Gradient of :func:`embedding` with respect to its table: [V, D] with
    ``scale * sum of dY[i] over tokens[i] == v`` in row v.

    dY: [*tokens.shape, D] fp32, bf16 or fp16.  The result has ``dtype``: dY's
    (the default) or fp32.  ``out`` ([V, D], rows at any stride) is written
    instead of a new tensor; with ``accumulate`` the gradient is added to what
    it holds, and only the rows of tokens in the batch are touched."""
    R.no_grad_of("embedding_grad", dY, out)
    V = int(V)
    if V < 1:
        raise ValueError(f"V must be positive, got {V}")
    if dY.dim() != tokens.dim() + 1 or dY.shape[:-1] != tokens.shape:
        raise ValueError(f"dY must be {tuple(tokens.shape)} + (D,), got {tuple(dY.shape)}")
    D, n = dY.shape[-1], tokens.numel()
    dev = dY.device
    if tokens.device != dev:
        R.same_device(dev, tokens=tokens)
    gpu = dY.is_cuda or not R.on_cpu(dY)
    dy = R.matrix(dY if dY.dim() == 2 else dY.reshape(n, D), "dY")
    tok = R.token_ids(tokens)
    scale = _scale(scale)
    if dtype is None:
        dtype = out.dtype if out is not None else dy.dtype
    if dtype not in (dy.dtype, torch.float32):
        raise ValueError(f"dtype must be dY's ({dy.dtype}) or float32, got {dtype}")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the out that it adds to")
        out = torch.empty(V, D, dtype=dtype, device=dev)
    else:
        R.output(out, (V, D), dtype, dev)
        R.apart(out, dy, "dY", in_place=False)
    if D == 0:
        return out
    at_dy, at_tok, at_out = dy.data_ptr() or null(dy), tok.data_ptr() or null(tok), out.data_ptr() or null(out)
    if not gpu:
        g, t = dy.float().contiguous(), tok.to(torch.int64)
        acc = out.float().contiguous().clone() if accumulate else torch.zeros((V, D), dtype=torch.float32)
        _native.check(_native.host().spmm_cpu_embedding_grad(n, V, D, _native.ptr(g), _native.ptr(t), scale,
                                                             _native.ptr(acc), 0), "cpu_embedding_grad")
        out.copy_(acc)
        return out
    lib = _native.hip()
    bytes_ = lib.spmm_embedding_grad_ws(n, V, D, R.TYPES[dy.dtype], out.stride(0), accumulate)
    if bytes_ < 0:
        raise ValueError(f"embedding_grad does not take {n} tokens over {V} rows")
    with R.on(dev):
        ws = torch.empty(bytes_, dtype=torch.uint8, device=dev) if bytes_ else None
        _native.check(lib.spmm_embedding_grad(at_dy, dy.stride(0), R.TYPES[dy.dtype], at_tok, tok.dtype == torch.int64,
                                              n, V, D, scale, at_out, out.stride(0), R.TYPES[dtype], accumulate,
                                              ws.data_ptr() if bytes_ else None, bytes_, R.stream(dev)),
                      "embedding_grad")
    return out
