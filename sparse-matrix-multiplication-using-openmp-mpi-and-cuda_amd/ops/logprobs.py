"""Log-probabilities of given tokens, with entropy and the top alternatives.

For each row z of logits over a vocabulary and a temperature T, with
``q = softmax(z / T)``: ``ln q[token]``, the entropy ``-sum q ln q``, and the k
largest logits with their log-probabilities as a CSR matrix (n x V, k entries a
row), which :func:`ops.distill.distill_loss` takes as a teacher.

* Masked logits (-inf) have q = 0 and add nothing to the entropy.  A row of
  nothing else has q = 0 everywhere, entropy 0 and log-probabilities of -inf.
* The largest logits come first, the lower column first among equal ones (+0
  and -0 are equal, NaN is above all numbers); -inf ones are listed too.
* Token -1 is padding: its log-probability is 0 and has no gradient.  A token
  outside the vocabulary has NaN, and so has its row's gradient.
* A NaN or +inf logit makes its row's results NaN.
* Sums are held in fp32; results are the same in every run.

gfx950 kernels: ``csrc/kernels/vocab_logits.hip``; CPU tensors use the OpenMP
kernels of ``csrc/host/vocab_cpu.cpp``.  Nothing here waits for the GPU, so
both directions can be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _native
from .._native import c_vp, null
from . import rows as R
from .csr import CSR

_native.register_hip("spmm_vocab_ws", C.c_int64, C.c_int64, C.c_int, C.c_int, restype=C.c_int64)
_native.register_hip("spmm_token_logprobs", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, C.c_int, C.c_int,
                     C.c_float, C.c_float, c_vp, c_vp, c_vp, c_vp, c_vp, C.c_int64, c_vp)
_native.register_hip("spmm_token_logprobs_grad", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, C.c_int,
                     C.c_float, C.c_float, c_vp, c_vp, c_vp, c_vp, C.c_int64, c_vp)

MAX_TOP = 128   # vocab_logits.hip kMaxTop
KEPT = 1 << 16  # bytes of workspace that live on with the result, which saves an allocation of 1.8 us
LOG2E = 1.0 / math.log(2.0)


@dataclass
class TokenLogprobs:
    logprob: torch.Tensor    # fp32 [n]
    entropy: torch.Tensor    # fp32 [n]
    stat: torch.Tensor       # fp32 [>= 4, n]: both, the row's maximum m and its sum of exp((z - m) / T); workspace
    temperature: float
    top: Optional[CSR]       # n x V, k entries a row, largest first (fp32 log-probabilities)


def logits_rows(logits: torch.Tensor) -> torch.Tensor:
    z = R.matrix(logits, "logits")
    if z.shape[1] < 1 or z.shape[1] >= 2 ** 31 - 4096:
        raise ValueError(f"a vocabulary has 1 to 2^31 - 4097 columns, got {z.shape[1]}")
    return z


def gradient_out(out: Optional[torch.Tensor], z: torch.Tensor) -> torch.Tensor:
    """A new gradient of z's shape and type, or the caller's (z itself allowed)."""
    if out is None:
        return torch.empty(*z.shape, dtype=z.dtype, device=z.device)
    R.output(out, z.shape, z.dtype, z.device)
    R.apart(out, z, "logits", in_place=True)
    return out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log-probability of ``tokens[i]`` (int32 or int64, [n]) in row i of
    ``logits`` ([n, V] fp32, bf16 or fp16, rows at any stride), the row's
    entropy, and its ``k`` (at most 128 and at most V; 0: none) largest logits."""
    R.no_grad_of("token_logprobs_grad", logits)
    z = logits_rows(logits)
    n, V = z.shape
    dev = z.device
    if tokens.device != dev:
        R.same_device(dev, tokens=tokens)
    if tokens.dim() != 1 or tokens.shape[0] != n:
        raise ValueError(f"tokens must be [{n}], got {tuple(tokens.shape)}")
    tok = R.token_ids(tokens)
    inv_t = R.inverse_temperature(temperature)
    k = int(k)
    if not 0 <= k <= min(MAX_TOP, V):
        raise ValueError(f"k must be between 0 and {min(MAX_TOP, V)}, got {k}")
    on_gpu = z.is_cuda or not R.on_cpu(z)
    gpu = on_gpu and n > 0
    bytes_ = _native.hip().spmm_vocab_ws(n, V, R.TYPES[z.dtype], k) if gpu else 0
    kept = bytes_ <= KEPT   # (a row's workspace is whole floats, and starts at 16 bytes)
    stat = torch.empty(4 + (bytes_ // (4 * n) if gpu and kept else 0), n, dtype=torch.float32, device=dev)
    logprob, entropy = stat[0], stat[1]
    top = None
    if k:
        top = CSR(n, V, torch.empty(n + 1, dtype=torch.int64, device=dev),
                  torch.empty(n * k, dtype=torch.int32, device=dev),
                  torch.empty(n * k, dtype=torch.float32, device=dev))
        if n == 0:
            top.rowptr.zero_()
        elif not on_gpu:
            torch.arange(0, n * k + 1, k, out=top.rowptr)
    res = TokenLogprobs(logprob, entropy, stat, float(temperature), top)
    if n == 0:
        return res
    at_z, at_tok, at_stat = z.data_ptr() or null(z), tok.data_ptr() or null(tok), stat.data_ptr() or null(stat)
    at = (top.rowptr.data_ptr(), top.col.data_ptr(), top.val.data_ptr()) if k else (None, None, None)
    if not on_gpu:
        zf, t = z.float().contiguous(), tok.to(torch.int64)
        _native.check(_native.host().spmm_cpu_token_logprobs(n, V, _native.ptr(zf), _native.ptr(t), inv_t, k, at_stat,
                                                             at[1], at[2], 0), "cpu_token_logprobs")
        return res
    with R.on(dev):
        ws = None if kept else torch.empty(bytes_, dtype=torch.uint8, device=dev)
        _native.check(_native.hip().spmm_token_logprobs(
            at_z, z.stride(0), n, V, R.TYPES[z.dtype], at_tok, tok.dtype == torch.int64, k,
            LOG2E * inv_t, inv_t, at_stat, *at, at_stat + 16 * n if kept else ws.data_ptr(), bytes_,
            R.stream(dev)), "token_logprobs")
    return res


def token_logprobs_grad(logits: torch.Tensor, tokens: torch.Tensor, stats: TokenLogprobs,
                        g_logprob: Optional[torch.Tensor] = None, g_entropy: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient with respect to the logits of ``sum_i g_logprob[i] logprob[i] +
    g_entropy[i] entropy[i]`` (fp32 [n], either may be absent), of the logits'
    shape and type.  ``stats``: what :func:`token_logprobs` returned for the
    same logits and tokens.  ``out`` may be the logits themselves.  A row with
    neither a log-probability's nor an entropy's gradient is zero and its
    logits are not read."""
    R.no_grad_of("token_logprobs_grad", logits, stats.stat, g_logprob, g_entropy, out)
    z = logits_rows(logits)
    gpu = z.is_cuda or not R.on_cpu(z)
    n, V = z.shape
    dev = z.device
    R.same_device(dev, tokens=tokens, g_logprob=g_logprob, g_entropy=g_entropy, stats=stats.stat)
    if tokens.dim() != 1 or tokens.shape[0] != n:
        raise ValueError(f"tokens must be [{n}], got {tuple(tokens.shape)}")
    stat = stats.stat
    if stat.dtype != torch.float32 or stat.dim() != 2 or stat.shape[0] < 4:
        raise ValueError(f"stats must be fp32 [4, {n}], got {stat.dtype} {tuple(stat.shape)}")
    if stat.shape[1] != n:
        raise ValueError(f"stats are of {stat.shape[1]} rows, the logits have {n}")
    stat = R.contiguous(stat)   # (some of a larger batch's rows)
    tok = R.token_ids(tokens)
    g, h = R.per_row(g_logprob, n, "g_logprob"), R.per_row(g_entropy, n, "g_entropy")
    inv_t = R.inverse_temperature(stats.temperature)
    out = gradient_out(out, z)
    if n == 0:
        return out
    at_z, at_tok, at_stat = z.data_ptr() or null(z), tok.data_ptr() or null(tok), stat.data_ptr() or null(stat)
    at_out = out.data_ptr() or null(out)
    at_g = g.data_ptr() or null(g) if g is not None else None
    at_h = h.data_ptr() or null(h) if h is not None else None
    if not gpu:
        zf, t = z.float().contiguous(), tok.to(torch.int64)
        acc = torch.empty((n, V), dtype=torch.float32)
        _native.check(_native.host().spmm_cpu_token_logprobs_grad(n, V, _native.ptr(zf), _native.ptr(t), inv_t,
                                                                  at_stat, at_g, at_h, _native.ptr(acc), 0),
                      "cpu_token_logprobs_grad")
        out.copy_(acc)
        return out
    with R.on(dev):
        _native.check(_native.hip().spmm_token_logprobs_grad(
            at_z, z.stride(0), n, V, R.TYPES[z.dtype], at_tok, tok.dtype == torch.int64, LOG2E * inv_t, inv_t, at_stat,
            at_g, at_h, at_out, out.stride(0), R.stream(dev)), "token_logprobs_grad")
    return out
