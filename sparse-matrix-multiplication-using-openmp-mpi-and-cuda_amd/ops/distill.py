"""Distillation from a teacher's top logits, forward and backward.

The teacher is a CSR matrix T (tokens x vocabulary): the logits or
log-probabilities that it stored for each token, in any order, any number a
row -- e.g. ``token_logprobs(...).top``.  With temperature tau,
``p = softmax(row of T / tau)`` over the stored entries and
``q = softmax(student's row / tau)`` over the whole vocabulary:

    loss  = sum_k p_k (ln p_k - ln q[c_k])
    dz_j  = weight (q_j - p_j) / tau

* A row without entries, without mass (all -inf) or of weight 0 has a zero
  gradient; without entries or mass its loss is 0 too.
* Column -1 marks an absent entry (a row padded to a fixed length); entries of
  equal columns add up.  A column outside the vocabulary, or a value of NaN or
  +inf, makes its row NaN.
* Masked student logits (-inf) have q = 0: the loss is +inf where the teacher
  has mass there.
* Sums are held in fp32; results are the same in every run.

gfx950 kernels: ``csrc/kernels/vocab_logits.hip``; CPU tensors use the OpenMP
kernel of ``csrc/host/vocab_cpu.cpp``.  Nothing here waits for the GPU, so
all three calls can be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _native
from .._native import c_vp, null
from . import rows as R
from .csr import CSR
from .logprobs import LOG2E, gradient_out, logits_rows

_native.register_hip("spmm_distill", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, c_vp, c_vp, C.c_int,
                     C.c_int64, C.c_float, C.c_float, c_vp, c_vp, c_vp, c_vp, c_vp, C.c_int64, c_vp, C.c_int64, c_vp)
_native.register_hip("spmm_distill_grad", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, c_vp, c_vp, C.c_int,
                     C.c_int64, C.c_float, C.c_float, c_vp, c_vp, c_vp, c_vp, C.c_int64, c_vp)


@dataclass
class DistillLoss:
    loss: torch.Tensor       # fp32 [n], a part of `saved` (clone it to keep it alone)
    saved: torch.Tensor      # fp32: loss; per row the student's maximum and sum, the teacher's two; the student's
                             # logits at the teacher's entries; workspace
    rows: int
    entries: int
    temperature: float


def _operands(logits: torch.Tensor, teacher: CSR):
    z = logits_rows(logits)
    n, V = z.shape
    ptr, col, val = teacher.rowptr, teacher.col, teacher.val
    if teacher.m != n or teacher.n != V:
        raise ValueError(f"the teacher is {teacher.m} x {teacher.n}, the logits {n} x {V}")
    dev = z.device
    if ptr.device != dev or col.device != dev or val.device != dev:
        R.same_device(dev, teacher=ptr, teacher_col=col, teacher_val=val)
    if ptr.dtype != torch.int64 or ptr.dim() != 1 or ptr.shape[0] != n + 1:
        raise ValueError(f"teacher.rowptr must be int64 [{n + 1}], got {ptr.dtype} {tuple(ptr.shape)}")
    if col.dtype != torch.int32 or col.dim() != 1:
        raise ValueError(f"teacher.col must be int32 [nnz], got {col.dtype} {tuple(col.shape)}")
    if val.dtype not in R.TYPES or val.shape != col.shape:
        raise ValueError(f"teacher.val must be float32, bfloat16 or float16 [{col.shape[0]}], got {val.dtype} "
                         f"{tuple(val.shape)}")
    return z, n, V, R.contiguous(ptr), R.contiguous(col), R.contiguous(val)


def _run(logits, teacher, weight, temperature, out, gradient) -> Tuple[DistillLoss, Optional[torch.Tensor]]:
    R.no_grad_of("distill_loss_grad", logits, weight, out, teacher.val)
    z, n, V, ptr, col, val = _operands(logits, teacher)
    dev, nnz, code = z.device, col.shape[0], R.TYPES[z.dtype]
    if weight is not None:
        R.same_device(dev, weight=weight)
        weight = R.per_row(weight, n, "weight")
    inv_t = R.inverse_temperature(temperature)
    gpu = z.is_cuda or not R.on_cpu(z)
    ws = _native.hip().spmm_vocab_ws(n, V, code, -1) if gpu else 0
    head = (5 * n + nnz + 3) // 4 * 4   # (the workspace starts at 16 bytes)
    saved = torch.empty(head + ws // 4, dtype=torch.float32, device=dev)
    res = DistillLoss(saved[:n], saved, n, nnz, float(temperature))
    if gradient:
        out = gradient_out(out, z)
    if n == 0:
        return res, out
    at, at_z, at_ptr = saved.data_ptr() or null(saved), z.data_ptr() or null(z), ptr.data_ptr() or null(ptr)
    at_col, at_val = col.data_ptr() or null(col), val.data_ptr() or null(val)
    w = weight.data_ptr() or null(weight) if weight is not None else None
    at_out = out.data_ptr() or null(out) if gradient else None
    if not gpu:
        zf, vf = z.float().contiguous(), val.float()
        acc = torch.empty((n, V), dtype=torch.float32) if gradient else None
        _native.check(_native.host().spmm_cpu_distill(
            n, V, _native.ptr(zf), at_ptr, at_col, _native.ptr(vf), nnz, inv_t, at, at + 4 * n, w, _native.ptr(acc), 0),
            "cpu_distill")
        if gradient:
            out.copy_(acc)
        return res, out
    with R.on(dev):
        _native.check(_native.hip().spmm_distill(
            at_z, z.stride(0), n, V, code, at_ptr, at_col, at_val, R.TYPES[val.dtype], nnz, LOG2E * inv_t, inv_t, at,
            at + 4 * n, at + 20 * n, w, at_out, out.stride(0) if gradient else 0, at + 4 * head, ws,
            R.stream(dev)), "distill")
    return res, out


def distill_loss(logits: torch.Tensor, teacher: CSR, temperature: float = 1.0) -> DistillLoss:
    """The loss of every row of ``logits`` ([n, V] fp32, bf16 or fp16, rows at
    any stride) against ``teacher`` (n x V CSR; values fp32, bf16 or fp16)."""
    return _run(logits, teacher, None, temperature, None, False)[0]


def distill_loss_grad(logits: torch.Tensor, teacher: CSR, weight: Optional[torch.Tensor] = None,
                      temperature: float = 1.0,
                      out: Optional[torch.Tensor] = None) -> Tuple[DistillLoss, torch.Tensor]:
    """Loss of every row and, in the same call, the gradient of ``sum_i
    weight[i] loss[i]`` (fp32 [n]; absent: 1) with respect to the logits, of
    their shape and type.  ``out`` may be the logits themselves."""
    return _run(logits, teacher, weight, temperature, out, True)


def distill_grad(logits: torch.Tensor, teacher: CSR, stats: DistillLoss, weight: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient alone, where the rows' weights are known only after the
    loss: ``stats`` is what :func:`distill_loss` returned for the same logits
    and teacher.  ``out`` may be the logits themselves."""
    R.no_grad_of("distill_grad", logits, stats.saved, weight, out, teacher.val)
    z, n, V, ptr, col, val = _operands(logits, teacher)
    dev, nnz = z.device, col.shape[0]
    R.same_device(dev, weight=weight, stats=stats.saved)
    weight = R.per_row(weight, n, "weight")
    if stats.rows != n or stats.entries != nnz:
        raise ValueError(f"stats are of {stats.rows} rows and {stats.entries} entries, the operands have {n} and {nnz}")
    inv_t = R.inverse_temperature(stats.temperature)
    saved = stats.saved
    if saved.dtype != torch.float32 or saved.dim() != 1 or saved.shape[0] < 5 * n + nnz:
        raise ValueError(f"stats.saved must be fp32 [{5 * n + nnz}] or longer, got {saved.dtype} {tuple(saved.shape)}")
    saved = R.contiguous(saved)
    out = gradient_out(out, z)
    if n == 0:
        return out
    if not z.is_cuda and R.on_cpu(z):
        return _run(z, teacher, weight, stats.temperature, out, True)[1]
    at, at_z, at_ptr = saved.data_ptr() or null(saved), z.data_ptr() or null(z), ptr.data_ptr() or null(ptr)
    at_col, at_val, at_out = col.data_ptr() or null(col), val.data_ptr() or null(val), out.data_ptr() or null(out)
    w = weight.data_ptr() or null(weight) if weight is not None else None
    with R.on(dev):
        _native.check(_native.hip().spmm_distill_grad(
            at_z, z.stride(0), n, V, R.TYPES[z.dtype], at_ptr, at_col, at_val, R.TYPES[val.dtype], nnz, LOG2E * inv_t,
            inv_t, at + 4 * n, at + 20 * n, w, at_out, out.stride(0), R.stream(dev)), "distill_grad")
    return out
