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
from .._native import c_vp
from . import rows as R
from .csr import CSR
from .logprobs import LOG2E, gradient_out, logits_rows

_native.register_hip("spmm_distill", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, c_vp, c_vp, C.c_int,
                     C.c_int64, C.c_float, C.c_float, c_vp, c_vp, c_vp, c_vp, c_vp, C.c_int64, c_vp, C.c_int64, c_vp)
_native.register_hip("spmm_distill_grad", c_vp, C.c_int64, C.c_int64, C.c_int64, C.c_int, c_vp, c_vp, c_vp, C.c_int,
                     C.c_int64, C.c_float, C.c_float, c_vp, c_vp, c_vp, c_vp, C.c_int64, c_vp)


@dataclass
class DistillLoss:
    loss: torch.Tensor       # fp32 [n]
    stat: torch.Tensor       # fp32 [n, 4]: student's maximum m and sum of exp((z - m) / tau), the teacher's two
    picked: torch.Tensor     # fp32 [nnz]: the student's logits at the teacher's entries
    temperature: float


def _operands(logits: torch.Tensor, teacher: CSR) -> Tuple[torch.Tensor, torch.Tensor]:
    z = logits_rows(logits)
    n, V = z.shape
    if teacher.m != n or teacher.n != V:
        raise ValueError(f"the teacher is {teacher.m} x {teacher.n}, the logits {n} x {V}")
    R.same_device(z.device, **{"teacher.rowptr": teacher.rowptr, "teacher.col": teacher.col, "teacher.val": teacher.val})
    if teacher.rowptr.dtype != torch.int64 or tuple(teacher.rowptr.shape) != (n + 1,):
        raise ValueError(f"teacher.rowptr must be int64 [{n + 1}], got {teacher.rowptr.dtype} "
                         f"{tuple(teacher.rowptr.shape)}")
    if teacher.col.dtype != torch.int32 or teacher.col.dim() != 1:
        raise ValueError(f"teacher.col must be int32 [nnz], got {teacher.col.dtype} {tuple(teacher.col.shape)}")
    if teacher.val.dtype not in R.TYPES or teacher.val.shape != teacher.col.shape:
        raise ValueError(f"teacher.val must be float32, bfloat16 or float16 [{teacher.nnz}], got {teacher.val.dtype} "
                         f"{tuple(teacher.val.shape)}")
    return z, CSR(n, V, teacher.rowptr.contiguous(), teacher.col.contiguous(), teacher.val.contiguous())


def _run(logits, teacher, weight, temperature, out, gradient) -> Tuple[DistillLoss, Optional[torch.Tensor]]:
    R.no_grad_of("distill_loss_grad", logits, weight, out, teacher.val)
    z, t = _operands(logits, teacher)
    n, V = z.shape
    dev = z.device
    R.same_device(dev, weight=weight)
    weight = R.per_row(weight, n, "weight")
    inv_t = R.inverse_temperature(temperature)
    loss = torch.empty(n, dtype=torch.float32, device=dev)
    stat = torch.empty((n, 4), dtype=torch.float32, device=dev)
    picked = torch.empty(t.nnz, dtype=torch.float32, device=dev)
    if gradient:
        out = gradient_out(out, z)
    res = DistillLoss(loss, stat, picked, float(temperature))
    if n == 0:
        return res, out
    P = _native.ptr
    if dev.type != "cuda":
        zf, val = z.float().contiguous(), t.val.float()
        acc = torch.empty((n, V), dtype=torch.float32) if gradient else None
        _native.check(_native.host().spmm_cpu_distill(n, V, P(zf), P(t.rowptr), P(t.col), P(val), t.nnz, inv_t, P(loss),
                                                      P(stat), P(weight), P(acc), 0), "cpu_distill")
        if gradient:
            out.copy_(acc)
        return res, out
    lib = _native.hip()
    code = R.TYPES[z.dtype]
    bytes_ = lib.spmm_vocab_ws(n, V, code, 0)
    with R.on(dev):
        ws = torch.empty(bytes_, dtype=torch.uint8, device=dev)
        _native.check(lib.spmm_distill(
            P(z), z.stride(0), n, V, code, P(t.rowptr), P(t.col), P(t.val), R.TYPES[t.val.dtype], t.nnz, LOG2E * inv_t,
            inv_t, P(loss), P(stat), P(picked), P(weight), P(out) if gradient else None,
            out.stride(0) if gradient else 0, P(ws), bytes_, _native.stream_ptr(dev)), "distill")
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
    R.no_grad_of("distill_grad", logits, weight, out, teacher.val)
    z, t = _operands(logits, teacher)
    n, V = z.shape
    dev = z.device
    R.same_device(dev, weight=weight, stats=stats.stat)
    weight = R.per_row(weight, n, "weight")
    if stats.stat.shape[0] != n or stats.picked.shape[0] != t.nnz:
        raise ValueError(f"stats are of {stats.stat.shape[0]} rows and {stats.picked.shape[0]} entries, the operands "
                         f"have {n} and {t.nnz}")
    inv_t = R.inverse_temperature(stats.temperature)
    out = gradient_out(out, z)
    if n == 0:
        return out
    P = _native.ptr
    if dev.type != "cuda":
        return _run(z, t, weight, stats.temperature, out, True)[1]
    with R.on(dev):
        _native.check(_native.hip().spmm_distill_grad(
            P(z), z.stride(0), n, V, R.TYPES[z.dtype], P(t.rowptr), P(t.col), P(t.val), R.TYPES[t.val.dtype], t.nnz,
            LOG2E * inv_t, inv_t, P(stats.stat), P(stats.picked), P(weight), P(out), out.stride(0),
            _native.stream_ptr(dev)), "distill_grad")
    return out
