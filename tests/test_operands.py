"""What the operators on rows over a vocabulary, and the products beside them,
refuse because a native call would go wrong on it without a word, and calls of
theirs that take a path of their own."""
import dataclasses
import math

import pytest
import torch
from torch.autograd import forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

import spmm_amd  # noqa: F401
from spmm_amd.ops.csr import CSR
from spmm_amd.ops.distill import distill_grad, distill_loss, distill_loss_grad
from spmm_amd.ops.embedding import embedding, embedding_grad
from spmm_amd.ops.logprobs import token_logprobs, token_logprobs_grad
from spmm_amd.ops.spmm import spmm

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


class Operands:
    """Small operands of all entry points, and each of these as a call of some of them."""

    def __init__(self, dev, dtype=torch.float32):
        g = torch.Generator().manual_seed(3)
        self.W = torch.randn(7, 9, generator=g).to(dtype).to(dev)
        self.dY = torch.randn(3, 9, generator=g).to(dtype).to(dev)
        self.z = torch.randn(3, 7, generator=g).to(dtype).to(dev)
        self.tok = torch.tensor([1, 6, 0], device=dev)
        self.g = torch.randn(3, generator=g).to(dev)
        self.w = torch.rand(3, generator=g).to(dev)
        self.T = CSR(3, 7, torch.tensor([0, 2, 2, 5], device=dev),
                     torch.tensor([1, 4, 0, 3, 6], dtype=torch.int32, device=dev),
                     torch.randn(5, generator=g).to(dev))

    def change(self, f):
        """The same with f applied to every floating-point operand."""
        o = object.__new__(Operands)
        o.tok = self.tok
        for name in ("W", "dY", "z", "g", "w"):
            setattr(o, name, f(getattr(self, name)))
        o.T = self.T.with_values(f(self.T.val))
        return o


CALLS = {
    "embedding": lambda o: embedding(o.W, o.tok, scale=1.5),
    "embedding_grad": lambda o: embedding_grad(o.dY, o.tok, 7, scale=1.5),
    "token_logprobs": lambda o: token_logprobs(o.z, o.tok, k=2),
    "token_logprobs_grad": lambda o: token_logprobs_grad(o.z, o.tok, token_logprobs(o.z, o.tok), o.g, o.w),
    "distill_loss": lambda o: distill_loss(o.z, o.T),
    "distill_loss_grad": lambda o: distill_loss_grad(o.z, o.T, o.w),
    "distill_grad": lambda o: distill_grad(o.z, o.T, distill_loss(o.z, o.T), o.w),
}


# ---- tensors without memory of their own ----------------------------------------------------------------------------

class Wrapper(torch.Tensor):
    """A subclass that holds another tensor and no memory itself."""

    @staticmethod
    def __new__(cls, x):
        r = torch.Tensor._make_wrapper_subclass(cls, x.shape, dtype=x.dtype, device=x.device, strides=x.stride())
        r.inner = x
        return r

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        out = func(*[a.inner if isinstance(a, Wrapper) else a for a in args], **(kwargs or {}))
        return Wrapper(out) if isinstance(out, torch.Tensor) else out


MEMORYLESS = {
    "meta": lambda x: x.to("meta"),
    "fake": lambda x: FakeTensorMode().from_tensor(x),
    "zero": lambda x: torch._efficientzerotensor(x.shape, dtype=x.dtype, device=x.device),
    "wrapper": Wrapper,
}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", MEMORYLESS)
@pytest.mark.parametrize("name", CALLS)
def test_tensors_without_memory_are_refused(dev, kind, name):
    o = Operands(dev).change(MEMORYLESS[kind])
    with pytest.raises(ValueError, match="no memory|on the CPU or a GPU|is on"):
        CALLS[name](o)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kind", MEMORYLESS)
def test_single_operands_without_memory_are_refused(dev, kind):
    f, o = MEMORYLESS[kind], Operands(dev)
    r, s = token_logprobs(o.z, o.tok), distill_loss(o.z, o.T)
    T = [CSR(3, 7, f(o.T.rowptr), o.T.col, o.T.val), CSR(3, 7, o.T.rowptr, f(o.T.col), o.T.val),
         CSR(3, 7, o.T.rowptr, o.T.col, f(o.T.val))]
    calls = [lambda: embedding(o.W, f(o.tok)), lambda: embedding(o.W, o.tok, out=f(o.dY)),
             lambda: embedding_grad(o.dY, f(o.tok), 7), lambda: embedding_grad(o.dY, o.tok, 7, out=f(o.W)),
             lambda: token_logprobs(o.z, f(o.tok)), lambda: token_logprobs_grad(o.z, o.tok, r, f(o.g)),
             lambda: token_logprobs_grad(o.z, o.tok, r, None, f(o.g)),
             lambda: token_logprobs_grad(o.z, o.tok, r, o.g, out=f(o.z)),
             lambda: distill_loss_grad(o.z, o.T, weight=f(o.w)), lambda: distill_loss_grad(o.z, o.T, out=f(o.z)),
             lambda: distill_grad(o.z, o.T, s, weight=f(o.w))]
    calls += [lambda t=t: distill_loss(o.z, t) for t in T]
    for call in calls:
        with pytest.raises(ValueError, match="no memory|is on|overlap"):
            call()


@pytest.mark.parametrize("kind", MEMORYLESS)
def test_products_of_tensors_without_memory_are_refused(kind):
    f, o = MEMORYLESS[kind], Operands("cpu")
    X = torch.randn(7, 128)
    for A, x in ((o.T.with_values(f(o.T.val)), X), (CSR(3, 7, f(o.T.rowptr), o.T.col, o.T.val), X), (o.T, f(X))):
        with pytest.raises(ValueError, match="no memory"):
            spmm(A, x)


# ---- tracers --------------------------------------------------------------------------------------------------------

def traced(how, f, x):
    if how == "jit":
        return torch.jit.trace(f, (x,), check_trace=False)
    if how == "fake mode":
        with FakeTensorMode(allow_non_fake_inputs=True):
            return f(x)
    kwargs = {"make_fx": {}, "fake": {"tracing_mode": "fake"}, "symbolic": {"tracing_mode": "symbolic"},
              "pre-dispatch": {"pre_dispatch": True}}[how]
    return make_fx(f, **kwargs)(x)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("how", ["jit", "make_fx", "fake", "symbolic", "pre-dispatch", "fake mode"])
@pytest.mark.parametrize("name", CALLS)
def test_tracers_are_refused(dev, how, name):
    """They record the allocation of the output and nothing of the kernel: what they return gives garbage."""
    o = Operands(dev)

    def call(z):
        r = CALLS[name](o.change(lambda x: z if x is o.z else x))
        r = r[1] if isinstance(r, tuple) else r
        return r if isinstance(r, torch.Tensor) else r.logprob if name == "token_logprobs" else r.loss

    with pytest.raises(ValueError, match="tracer"):
        traced(how, call, o.z)


@pytest.mark.parametrize("dev", DEVICES)
def test_modes_that_record_nothing_are_taken(dev):
    o = Operands(dev)
    want = token_logprobs(o.z, o.tok).logprob
    with torch.device(dev), FlopCounterMode(display=False), torch.inference_mode():
        assert torch.equal(token_logprobs(o.z, o.tok).logprob, want)
    assert torch.equal(token_logprobs(o.z, o.tok).logprob, want)


def test_compiled_callers_run_the_operators():
    """torch.compile leaves a caller's compiled parts at these calls and runs them as they are."""
    o = Operands("cpu")

    def step(z, tok):
        return token_logprobs(z + 1.0, tok).logprob * 2.0

    f = torch.compile(step, backend="eager")
    for z in (o.z, o.z * 3.0):
        assert torch.equal(f(z, o.tok), step(z, o.tok))


# ---- forward-mode differentiation -----------------------------------------------------------------------------------

@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(dev, dtype, name):
    o = Operands(dev, dtype)
    with forward_ad.dual_level():
        CALLS[name](o)                                        # tensors without a tangent
        dual = o.change(lambda x: forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            CALLS[name](dual)
        CALLS[name](dual.change(lambda x: forward_ad.unpack_dual(x).primal))
    CALLS[name](o)


@pytest.mark.parametrize("dev", DEVICES)
def test_each_tangent_is_refused(dev):
    o = Operands(dev)
    r, s = token_logprobs(o.z, o.tok), distill_loss(o.z, o.T)
    with forward_ad.dual_level():
        def d(x):
            return forward_ad.make_dual(x, torch.ones_like(x))

        calls = [lambda: embedding(o.W, o.tok, out=d(o.dY.clone())),
                 lambda: embedding_grad(o.dY, o.tok, 7, out=d(o.W.clone()), accumulate=True),
                 lambda: token_logprobs_grad(o.z, o.tok, r, d(o.g)),
                 lambda: token_logprobs_grad(o.z, o.tok, r, None, d(o.g)),
                 lambda: token_logprobs_grad(d(o.z), o.tok, r, o.g),
                 lambda: token_logprobs_grad(o.z, o.tok, dataclasses.replace(r, stat=d(r.stat)), o.g),
                 lambda: distill_loss_grad(o.z, o.T, weight=d(o.w)),
                 lambda: distill_loss(o.z, o.T.with_values(d(o.T.val))),
                 lambda: distill_grad(o.z, o.T, s, weight=d(o.w)),
                 lambda: distill_grad(o.z, o.T, dataclasses.replace(s, saved=d(s.saved)))]
        for call in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                call()


# ---- views that hold the negatives of their values ------------------------------------------------------------------

def held_negated(x):
    """x as the negative of what is in memory."""
    y = torch._neg_view(-x)
    assert y.is_neg() and torch.equal(y, x)
    return y


def results(r):
    """All tensors of a result."""
    if isinstance(r, torch.Tensor):
        return [r]
    if isinstance(r, tuple):
        return [t for x in r for t in results(x)]
    return [r.loss] if hasattr(r, "loss") else [r.logprob, r.entropy] + ([r.top.col, r.top.val] if r.top else [])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CALLS)
def test_negated_views_are_their_values(dev, dtype, name):
    o = Operands(dev, dtype)
    for got, want in zip(results(CALLS[name](o.change(held_negated))), results(CALLS[name](o)), strict=True):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dev", DEVICES)
def test_negated_tokens_and_statistics_are_their_values(dev):
    o = Operands(dev)
    tok, r, s = held_negated(o.tok), token_logprobs(o.z, o.tok), distill_loss(o.z, o.T)
    assert torch.equal(embedding(o.W, tok), o.W[o.tok])
    assert torch.equal(embedding_grad(o.dY, tok, 7), embedding_grad(o.dY, o.tok, 7))
    assert torch.equal(token_logprobs(o.z, tok).logprob, r.logprob)
    want = token_logprobs_grad(o.z, o.tok, r, o.g, o.w)
    assert torch.equal(token_logprobs_grad(o.z, tok, r, o.g, o.w), want)
    stat = held_negated(r.stat[:4].clone())
    assert torch.equal(token_logprobs_grad(o.z, o.tok, dataclasses.replace(r, stat=stat), o.g, o.w), want)
    want = distill_grad(o.z, o.T, s, o.w)
    saved = held_negated(s.saved[:5 * 3 + 5].clone())
    assert torch.equal(distill_grad(o.z, o.T, dataclasses.replace(s, saved=saved), o.w), want)
    T = CSR(3, 7, held_negated(o.T.rowptr), held_negated(o.T.col), o.T.val)
    assert torch.equal(distill_loss_grad(o.z, T, o.w)[1], want)


@pytest.mark.parametrize("dev", DEVICES)
def test_negated_outputs_are_refused(dev):
    o = Operands(dev)
    r, s = token_logprobs(o.z, o.tok), distill_loss(o.z, o.T)
    before = [x.clone() for x in (o.W, o.dY, o.z)]
    for call in (lambda: embedding(o.W, o.tok, out=torch._neg_view(o.dY)),
                 lambda: embedding_grad(o.dY, o.tok, 7, out=torch._neg_view(o.W)),
                 lambda: embedding_grad(o.dY, o.tok, 7, out=torch._neg_view(o.W), accumulate=True),
                 lambda: token_logprobs_grad(o.z, o.tok, r, o.g, out=torch._neg_view(o.z)),
                 lambda: distill_loss_grad(o.z, o.T, out=torch._neg_view(o.z)),
                 lambda: distill_grad(o.z, o.T, s, out=torch._neg_view(o.z))):
        with pytest.raises(ValueError, match="negative bit"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(before, (o.W, o.dY, o.z)))


def test_the_imaginary_part_of_a_conjugate():
    c = torch.randn(7, 9, dtype=torch.complex64, generator=torch.Generator().manual_seed(5))
    W, tok = c.conj().imag, torch.tensor([1, 6, 0])
    assert W.is_neg() and torch.equal(embedding(W, tok), -c.imag[tok])
    X = torch.randn(7, 128, generator=torch.Generator().manual_seed(6))
    A = Operands("cpu").T
    with pytest.raises(ValueError, match="negative bit"):
        spmm(A, torch._neg_view(X))


# ---- statistics of the distillation ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dev", DEVICES)
def test_statistics_that_are_not_the_losses_are_refused(dev):
    """The kernel reads 5 numbers a row and one an entry from them."""
    o = Operands(dev)
    s = distill_loss(o.z, o.T)
    want = distill_grad(o.z, o.T, s, o.w)
    for saved in (s.saved[:5 * 3 + 4], s.loss, s.saved.bfloat16(), s.saved.double(), s.saved[:16].view(4, 4)):
        with pytest.raises(ValueError, match="stats.saved must be"):
            distill_grad(o.z, o.T, dataclasses.replace(s, saved=saved), o.w)
    apart = torch.stack([s.saved, s.saved], dim=1)[:, 0]
    for saved in (s.saved[:5 * 3 + 5].clone(), apart):
        assert torch.equal(distill_grad(o.z, o.T, dataclasses.replace(s, saved=saved), o.w), want)
