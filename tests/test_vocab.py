"""Operators on rows over a vocabulary (embedding lookup and gradient, token
log-probabilities, distillation) against their definitions in 64 bits.

Tolerances count roundings.  A result of type t is off by at most half a step,
``finfo(t).eps / 2`` of its value (plus half the smallest subnormal step).  The
fp32 sums behind it add at most 256 terms one behind the other in a thread,
then at most 28 levels of threads, waves and segments: (256 + 28) 2^-24 of the
sum of magnitudes.  Each term exp2(u) is off by 2^-23 (the instruction) plus
|u| 2^-23 (u is rounded once, its factor log2(e) / T once): below 60 2^-24
weighted by the term, whose u above -30 alone counts.  SUM covers them.
"""
import dataclasses
import math

import pytest
import torch

import spmm_amd  # noqa: F401
from spmm_amd.ops.csr import CSR
from spmm_amd.ops.distill import distill_grad, distill_loss, distill_loss_grad
from spmm_amd.ops.embedding import embedding, embedding_grad
from spmm_amd.ops.logprobs import token_logprobs, token_logprobs_grad

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
SUM = 400 * U


def half_step(t, ref):
    """The most that rounding to type t changes ref."""
    f = torch.finfo(t)
    return ref.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def near(got, ref, tol):
    """got is within tol of ref wherever ref is a number, and equal to it elsewhere.  A number beyond the type of got
    (a logit of the type's lowest value, divided by a temperature below 1) rounds to infinity there."""
    beyond = ref.abs() > torch.finfo(got.dtype).max
    ref = torch.where(beyond, torch.sign(ref) * math.inf, ref)
    got, ref, tol = got.double().cpu(), ref.double().cpu(), torch.as_tensor(tol).double().cpu().expand_as(ref)
    assert got.shape == ref.shape
    fine = torch.isfinite(ref)
    assert torch.equal(got.isnan(), ref.isnan())
    odd = ~fine & ~ref.isnan()
    assert torch.equal(got[odd], ref[odd])
    off = (got - ref).abs()[fine] - tol[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{off.max().item():.3g} beyond the tolerance"


def gen(seed=0):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ---- embedding ------------------------------------------------------------------------------------------------------

def ref_lookup(W, tok, scale):
    t = tok.reshape(-1).cpu().long()
    V = W.shape[0]
    y = W.cpu().double()[t.clamp(0, V - 1)] * scale
    y[t == -1] = 0.0
    y[(t < -1) | (t >= V)] = math.nan
    return y.view(*tok.shape, W.shape[1])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,D,n", [(1, 1, 1), (7, 3, 5), (50, 8, 64), (50, 33, 65), (300, 64, 100), (1000, 257, 33),
                                   (100, 512, 17), (64, 1111, 40), (33, 2048, 70), (20, 4100, 9)])
def test_lookup(dev, dtype, V, D, n):
    g = gen(V + D)
    W = torch.randn(V, D, generator=g).to(dtype).to(dev)
    tok = torch.randint(0, V, (n,), generator=g)
    tok[::7] = -1
    for kind in (torch.int64, torch.int32):
        ref = ref_lookup(W, tok, 1.7)
        # two roundings in fp32 (the scale, the product), then the type's
        near(embedding(W, tok.to(kind).to(dev), scale=1.7), ref, half_step(dtype, ref) + 3 * U * ref.abs())


@pytest.mark.parametrize("dev", DEVICES)
def test_lookup_layouts(dev):
    g = gen(1)
    big = torch.randn(40, 50, generator=g).to(torch.bfloat16).to(dev)
    W = big[:, 3:36]                              # rows at a stride, starting in the middle of 16 bytes
    tok = torch.randint(0, 40, (3, 4), generator=g).to(dev)
    assert torch.equal(embedding(W, tok), W[tok])
    assert torch.equal(embedding(W, tok.t()), W[tok.t()])          # a transposed token matrix
    assert torch.equal(embedding(W, tok[0, 0]), W[tok[0, 0]])       # one token, no dimension
    assert torch.equal(embedding(W.t(), tok[:, 0] % 33), W.t()[tok[:, 0] % 33])   # columns that are not adjacent
    assert embedding(W, tok[:0]).shape == (0, 4, 33)
    out = torch.full((12, 40), 9.0, dtype=torch.bfloat16, device=dev)
    embedding(W, tok.reshape(-1), out=out[:, 2:35])
    assert torch.equal(out[:, 2:35], W[tok.reshape(-1)])
    assert (out[:, :2] == 9).all() and (out[:, 35:] == 9).all()
    odd = torch.tensor([0, -2, 40, 2 ** 40, -2 ** 40, -1], device=dev)
    y = embedding(W, odd)
    assert torch.equal(y[0], W[0]) and y[1:5].isnan().all() and (y[5] == 0).all()


def ref_grad(dY, tok, V, scale, start=None):
    """The gradient and the sum of magnitudes behind it."""
    t = tok.reshape(-1).cpu().long()
    d = dY.cpu().double().reshape(t.numel(), dY.shape[-1])
    keep = (t >= 0) & (t < V)
    zero = torch.zeros(V, dY.shape[-1], dtype=torch.float64)
    s = zero.index_add(0, t[keep], d[keep]) * scale
    mag = zero.index_add(0, t[keep], d[keep].abs()) * abs(scale)
    count = torch.bincount(t[keep], minlength=V).double()[:, None]
    if start is not None:
        s, mag = s + start.cpu().double(), mag + start.cpu().double().abs()
    return s, mag, count


def check_grad(dY, tok, V, scale, to, accumulate, dev, seed=0):
    out = None
    if accumulate:
        out = torch.randn(V, dY.shape[-1], generator=gen(seed + 5)).to(to).to(dev)
    ref, mag, count = ref_grad(dY, tok, V, scale, out)
    got = embedding_grad(dY.to(dev), tok.to(dev), V, scale=scale, dtype=to, out=None if out is None else out.clone(),
                         accumulate=accumulate)
    assert got.dtype == to
    # each of a row's additions rounds once, then the scale, its product and the accumulation do
    near(got, ref, half_step(to, ref) + (count + 4) * U * mag)
    if accumulate:   # rows without a token keep their bits
        rest = (count == 0)[:, 0]
        assert torch.equal(got.cpu()[rest], out.cpu()[rest])
    again = embedding_grad(dY.to(dev), tok.to(dev), V, scale=scale, dtype=to, out=None if out is None else out.clone(),
                           accumulate=accumulate)
    assert torch.equal(got, again)
    return got


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,to", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                      (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                      (torch.float16, torch.float32)])
@pytest.mark.parametrize("V,D,n", [(1, 1, 1), (1, 5, 100), (9, 8, 31), (9, 9, 33), (200, 70, 64), (17, 600, 300),
                                   (1000, 260, 65), (50, 1025, 129)])
def test_grad(dev, dtype, to, accumulate, V, D, n):
    g = gen(V * D + n)
    dY = torch.randn(n, D, generator=g).to(dtype)
    tok = torch.randint(0, V, (n,), generator=g)
    if n > 10:
        tok[::9] = -1
        tok[4], tok[5] = V, -7       # not in the table: no gradient
    check_grad(dY, tok, V, 0.3, to, accumulate, dev, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one token", "all padding", "sorted", "two runs"])
@pytest.mark.parametrize("n", [2047, 12288, 12289, 20000, 70001, 140000])
def test_grad_distributions(kind, n):
    """Both sorts, runs through many tiles, a whole batch of one token."""
    g = gen(n)
    V, D = 5000, 72
    tok = {"uniform": lambda: torch.randint(0, V, (n,), generator=g),
           "zipf": lambda: (V ** torch.rand(n, generator=g, dtype=torch.float64)).long().clamp_max(V - 1),
           "one token": lambda: torch.full((n,), 4321),
           "all padding": lambda: torch.full((n,), -1),
           "sorted": lambda: torch.arange(n) * V // n,
           "two runs": lambda: (torch.arange(n) > n // 3).long() * (V - 1)}[kind]()
    dY = torch.randn(n, D, generator=g).to(torch.bfloat16)
    check_grad(dY, tok, V, 1.0, torch.float32, False, "cuda")
    check_grad(dY, tok.to(torch.int32), V, 1.0, torch.bfloat16, True, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 1023, 1024, 1 << 20, (1 << 20) + 1, 3_000_000])
def test_grad_table_sizes(V):
    """One, two and three radix passes, key counts at powers of two."""
    g = gen(V)
    n, D = 10000, 12
    tok = torch.randint(0, V, (n,), generator=g)
    tok[0], tok[1], tok[2] = V - 1, -1, V
    check_grad(torch.randn(n, D, generator=g).to(torch.float16), tok, V, 2.0, torch.float32, False, "cuda")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 9, 8), (8, 5, 513), (9, 70, 64), (64, 2, 1000), (65, 4000, 33), (300, 1, 40),
                                   (1000, 100, 4100), (1024, 333, 72), (1025, 333, 72), (0, 40, 9)])
def test_grad_short_batches(dev, dtype, n, V, D):
    """Batches on both sides of what is summed without a sort, into tables with and without gaps between the rows."""
    g = gen(n + D)
    tok = torch.randint(-1, V + 1, (n,), generator=g)
    tok[: n // 3] = V - 1
    dY = torch.randn(n, D, generator=g).to(dtype)
    ref, mag, count = ref_grad(dY, tok, V, 1.25)
    tol = half_step(dtype, ref) + (count + 4) * U * mag
    for wide in (D, D + 24):
        table = torch.full((V + 1, wide), 7.0, dtype=dtype, device=dev)
        out = table[:V, :D]
        assert embedding_grad(dY.to(dev), tok.to(dev), V, scale=1.25, out=out) is out
        near(out, ref, tol)
        assert (table[V] == 7).all() and (table[:, D:] == 7).all()
    check_grad(dY, tok.to(torch.int32), V, 1.25, torch.float32, True, dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 4, 7])
def test_grad_narrow_rows_of_a_frequent_token(dev, dtype, D):
    g = gen(D)
    V, n = 37, 50001
    tok = torch.randint(-1, V + 1, (n,), generator=g)
    tok[torch.rand(n, generator=g) < 0.8] = 5
    dY = torch.randn(n, D, generator=g).to(dtype)
    check_grad(dY, tok, V, 0.5, dtype, False, dev)
    check_grad(dY, tok % 30, V, 0.5, torch.float32, True, dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_grad_layouts(dev):
    g = gen(2)
    V, D = 30, 20
    tok = torch.randint(0, V, (4, 6), generator=g)
    wide = torch.randn(4, 6, 2 * D, generator=g)
    dY = wide[..., 3:3 + D]
    ref, _, _ = ref_grad(dY, tok, V, 1.0)
    out = torch.full((V, D + 5), 7.0).to(dev)
    r = embedding_grad(dY.to(dev)[...], tok.to(dev), V, out=out[:, 1:1 + D])
    near(r, ref, 40 * U * ref.abs() + 1e-5)
    assert (out[:, 0] == 7).all() and (out[:, 1 + D:] == 7).all()
    none = embedding_grad(dY.to(dev)[:0], tok.to(dev)[:0], V)
    assert none.shape == (V, D) and (none == 0).all()
    keep = torch.randn(V, D, generator=g).to(dev)
    assert torch.equal(embedding_grad(dY.to(dev)[:0], tok.to(dev)[:0], V, out=keep.clone(), accumulate=True), keep)
    one = dY[0, 0].to(dev).expand(4, 6, D)       # a broadcast gradient
    near(embedding_grad(one, tok.to(dev), V), ref_grad(one.cpu(), tok, V, 1.0)[0], torch.tensor(1e-5))


@pytest.mark.parametrize("dev", DEVICES)
def test_grad_is_the_lookups(dev):
    """<dY, scale S W> = <scale S^T dY, W> on whole numbers, exactly, and differences of the lookup."""
    g = gen(3)
    V, D, n = 40, 24, 90
    W = torch.randint(-8, 9, (V, D), generator=g).float().to(dev)
    dY = torch.randint(-8, 9, (n, D), generator=g).float().to(dev)
    tok = torch.randint(-1, V, (n,), generator=g).to(dev)
    dW = embedding_grad(dY, tok, V, scale=2.0)
    assert (dY * embedding(W, tok, 2.0)).sum() == (dW * W).sum()
    step = torch.zeros_like(W)
    step[tok[5], 7] = 1.0
    assert (dY * (embedding(W + step, tok, 2.0) - embedding(W - step, tok, 2.0))).sum() / 2 == dW[tok[5], 7]


# ---- log-probabilities ----------------------------------------------------------------------------------------------

def ref_logprobs(z, T):
    """ln q, q, entropy in 64 bits; a row of -inf alone has q = 0."""
    z = z.cpu().double()
    m = z.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).amax(1, keepdim=True)
    t = (z - torch.where(m == -math.inf, 0.0, m)) / T
    s = t.exp().sum(1, keepdim=True)
    logq = t - torch.where(s == 0, 0.0, s.log())
    q = logq.exp()
    return logq, q, -torch.where(q == 0, 0.0, q * logq).sum(1)


def order_of(z, k):
    z = z.cpu().double() + 0.0
    rank = torch.where(z.isnan(), math.inf, z)
    # NaN above +inf: two stable sorts, the minor key first
    a = torch.sort(rank, dim=1, descending=True, stable=True).indices
    b = torch.sort(z.gather(1, a).isnan().to(torch.int8), dim=1, descending=True, stable=True).indices
    return a.gather(1, b)[:, :k]


def check_logprobs(z, tok, k, T, dev):
    n, V = z.shape
    r = token_logprobs(z.to(dev), tok.to(dev), k=k, temperature=T)
    logq, q, H = ref_logprobs(z, T)
    t = tok.cpu().long()
    lp = logq.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    lp = torch.where(t == -1, 0.0, lp)
    lp = torch.where((t < -1) | (t >= V), math.nan, lp)
    big = 1 + logq.abs().where(torch.isfinite(logq), torch.zeros(())).gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    near(r.logprob, lp, SUM + 8 * U * (big + math.log(V)))
    near(r.entropy, H, SUM * (1 + math.log(V)))
    if k:
        idx = order_of(z, k)
        assert r.top.m == n and r.top.n == V
        assert torch.equal(r.top.rowptr.cpu(), torch.arange(0, n * k + 1, k))
        assert torch.equal(r.top.col.view(n, k).cpu().long(), idx)
        val = logq.gather(1, idx)
        near(r.top.val.view(n, k), val,
             SUM + 8 * U * (val.abs().where(torch.isfinite(val), torch.zeros(())) + math.log(V)))
    else:
        assert r.top is None
    return r


def logits(n, V, dtype, seed=0):
    g = gen(seed + V)
    z = torch.randn(n, V, generator=g) * 3
    return z.to(dtype), torch.randint(0, V, (n,), generator=g)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V", [(1, 1), (3, 2), (5, 7), (2, 8), (4, 63), (3, 100), (2, 2047), (3, 2049), (2, 4097),
                                 (3, 8200), (2, 16384), (3, 16389), (2, 40001), (1, 131072)])
def test_logprobs(dev, dtype, n, V):
    z, tok = logits(n, V, dtype)
    for k in sorted({0, 1, min(V, 5), min(V, 64), min(V, 65), min(V, 128)}):
        check_logprobs(z, tok if k % 2 else tok.to(torch.int32), k, 1.0 if k else 0.7, dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 3000, 33001])
def test_logprobs_masks_and_ties(dev, dtype, V):
    z, tok = logits(12, V, dtype, seed=1)
    z[0] = 0.5                                    # all equal
    z[1] = -math.inf                              # nothing left
    z[2, 3:] = -math.inf                          # three left
    z[3] = torch.finfo(dtype).min                 # masked by the lowest value throughout
    z[4, 10:] = torch.finfo(dtype).min
    z[5] = torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0)
    z[6, V // 2] = math.nan
    z[7, V - 1] = math.inf
    z[8] = (z[8].float() * 0.5).round().to(dtype)  # many equal values
    z[9, :-1] = -math.inf
    z[10] = torch.linspace(-4, 4, V).to(dtype)     # ascending: every later logit is larger
    z[11] = z[11] * 0 + torch.finfo(dtype).max
    tok[2], tok[4], tok[9], tok[10] = 1, 2, V - 1, -1
    for k in (0, 3, 20, 50):
        check_logprobs(z, tok, k, 1.0, dev)
    check_logprobs(z[:, : V - 1].contiguous(), tok.clamp_max(V - 2), 40, 2.5, dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_long_rows_of_ties_and_infinities(dev, dtype):
    """More candidates than are ranked at once, fewer logits than alternatives, infinities beside other bits of a word."""
    V = 131072 + 3
    z, tok = logits(8, V, dtype, seed=5)
    z[0] = 1.25
    z[1] = -math.inf
    z[1, ::40000] = torch.tensor([1.0, -2.0, 3.0, 0.0]).to(dtype)
    z[2] = (z[2].float() * 0.25).round().to(dtype)
    z[3, 70001], z[3, 70000] = math.inf, -1.5
    z[4, 5], z[4, 4] = math.nan, -1.5
    z[5] = torch.linspace(-9, 9, V).to(dtype)
    z[6, :-2] = -math.inf
    z[7] = math.nan
    tok[1], tok[6] = 40000, V - 1
    for k in (1, 20, 64, 128):
        check_logprobs(z, tok, k, 1.0, dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V", [(1100, 500), (520, 16387), (300, 33003), (1030, 8199)])
def test_logprobs_many_rows(dtype, n, V):
    """More rows than are taken in one launch with their alternatives."""
    z, tok = logits(n, V, dtype, seed=44)
    z[:, ::3] = -math.inf
    z[5] = -math.inf
    z[6] = 1.0
    z[7, V // 2], z[8, 3] = math.nan, math.inf
    tok[::9] = -1
    check_logprobs(z, tok, 17, 1.3, "cuda")
    check_logprobs(z, tok, 0, 1.3, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_rows_of_millions(dtype):
    """More groups in a row than a wave keeps in registers."""
    V = 9_000_001
    z, tok = logits(2, V, dtype, seed=33)
    z[1, ::3] = 4.5
    for k in (2, 128):
        check_logprobs(z, tok, k, 1.0, "cuda")


@pytest.mark.gpu
def test_more_rows_than_workgroups():
    """Beyond the largest grid the workgroups go on with further rows: those have the results of a call of their own."""
    n, V, last = (1 << 23) + 777, 9, 1000
    z = torch.randn(n, V, generator=gen(34)).to(torch.bfloat16).cuda()
    tok = torch.randint(0, V, (n,), generator=gen(35)).cuda()
    g = torch.rand(n, generator=gen(36)).cuda()
    a, b = token_logprobs(z, tok, k=3), token_logprobs(z[-last:], tok[-last:], k=3)
    assert torch.equal(a.stat[:4, -last:], b.stat[:4])
    assert torch.equal(a.top.col[-3 * last:], b.top.col) and torch.equal(a.top.val[-3 * last:], b.top.val)
    dz = token_logprobs_grad(z, tok, a, g, g)
    assert torch.equal(dz[-last:], token_logprobs_grad(z[-last:], tok[-last:], b, g[-last:], g[-last:]))
    (la, da), (lb, db) = distill_loss_grad(z, a.top, g), distill_loss_grad(z[-last:], b.top, g[-last:])
    assert torch.equal(la.loss[-last:], lb.loss) and torch.equal(da[-last:], db)
    W = torch.randn(300, 520, generator=gen(37)).to(torch.bfloat16).cuda()
    y = embedding(W, tok)
    assert torch.equal(y[-last:], W[tok[-last:]])
    few = torch.randint(0, 1 << 27, (500,), generator=gen(38)).cuda()
    few[0] = (1 << 27) + 999
    dW, used = embedding_grad(y[:500, :8], few, (1 << 27) + 1000), few.unique()
    assert torch.equal(dW[used], embedding_grad(y[:500, :8], torch.searchsorted(used, few), used.numel()))
    dW[used] = 0
    assert torch.equal(dW, torch.zeros_like(dW))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [3, 700, 20001])
def test_logprobs_order_of_the_smallest(dev, dtype, V):
    """Logits of a few of the type's smallest steps around zero, of both signs."""
    f = torch.finfo(dtype)
    step = f.smallest_normal * f.eps
    z = (torch.randint(-3, 4, (4, V), generator=gen(24)).double() * step).to(dtype)
    z[1] = -z[1].abs()
    z[2, : V // 2] = -math.inf
    check_logprobs(z, torch.randint(0, V, (4,), generator=gen(25)), min(V, 100), 1.0, dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_logprobs_layouts(dev):
    z, tok = logits(6, 501, torch.bfloat16, seed=2)
    wide = torch.zeros(6, 600, dtype=torch.bfloat16, device=dev)
    wide[:, 37:538] = z.to(dev)
    a = token_logprobs(z.to(dev), tok.to(dev), k=9)
    for other in (wide[:, 37:538], z.t().contiguous().t().to(dev)):
        b = token_logprobs(other, tok.to(dev), k=9)
        assert torch.equal(a.logprob, b.logprob) and torch.equal(a.top.col, b.top.col)
    one = z[:1].to(dev).expand(6, 501)             # one row for all tokens
    c = token_logprobs(one, tok.to(dev))
    assert torch.equal(c.entropy, c.entropy[:1].expand(6))
    e = token_logprobs(z[:0].to(dev), tok[:0].to(dev), k=4)
    assert e.logprob.shape == (0,) and e.top.m == 0 and e.top.rowptr.tolist() == [0]
    odd = torch.tensor([-1, -2, 501, 2 ** 40, 0, 500], device=dev)
    d = token_logprobs(z.to(dev), odd).logprob
    assert d[0] == 0 and d[1:4].isnan().all() and d[4:].isfinite().all()


def check_token_grad(z, tok, g, h, T, dev, inplace=False):
    n, V = z.shape
    zd, td = z.clone().to(dev), tok.to(dev)
    r = token_logprobs(zd, td, temperature=T)
    got = token_logprobs_grad(zd, td, r, None if g is None else g.to(dev), None if h is None else h.to(dev),
                              out=zd if inplace else None)
    assert got.dtype == z.dtype
    logq, q, H = ref_logprobs(z, T)
    t = tok.cpu().long()
    gg = torch.zeros(n, dtype=torch.float64) if g is None else g.double()
    gg = torch.where(t == -1, 0.0, gg)
    hh = torch.zeros(n, dtype=torch.float64) if h is None else h.double()
    hot = torch.zeros(n, V, dtype=torch.float64)
    ok = (t >= 0) & (t < V)
    hot[ok, t[ok]] = 1.0
    qlogq = torch.where(q == 0, 0.0, q * logq)
    ref = (gg[:, None] * (hot - q) - hh[:, None] * (qlogq + q * H[:, None])) / T
    ref[(gg == 0) & (hh == 0)] = 0.0
    ref[(t < -1) | (t >= V)] = math.nan
    mag = (gg.abs()[:, None] * (hot + q) + hh.abs()[:, None] * (qlogq.abs() + q * (H.abs()[:, None] + 1 + math.log(V)))) / T
    near(got, ref, half_step(z.dtype, ref) + 2 * SUM * mag.nan_to_num(0.0) + half_step(z.dtype, torch.zeros(())))
    return got


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V", [(1, 1), (4, 9), (3, 100), (2, 2049), (3, 4100), (2, 8193), (2, 16385), (3, 33001)])
def test_logprobs_grad(dev, dtype, n, V):
    z, tok = logits(n, V, dtype, seed=3)
    g, h = torch.randn(n, generator=gen(4)), torch.randn(n, generator=gen(5))
    check_token_grad(z, tok, g, h, 1.0, dev)
    check_token_grad(z, tok, g, None, 0.7, dev)
    check_token_grad(z, tok, None, h, 2.0, dev, inplace=True)
    check_token_grad(z, tok, None, None, 1.0, dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_logprobs_grad_masks(dev):
    V = 3000
    z, tok = logits(8, V, torch.float32, seed=4)
    z[0] = -math.inf
    z[1, 5:] = -math.inf
    z[2] = torch.finfo(torch.float32).min
    z[3, 1:] = torch.finfo(torch.float32).min
    z[4] = math.nan
    tok[1], tok[3], tok[4], tok[5], tok[6] = 2, 0, -1, -1, V
    g, h = torch.randn(8, generator=gen(6)), torch.randn(8, generator=gen(7))
    h[4] = 0.0                       # a padded row of garbage: nothing flows, nothing is read
    got = check_token_grad(z, tok, g, h, 1.5, dev)
    assert (got[4] == 0).all() and got[6].isnan().all()


@pytest.mark.parametrize("dev", DEVICES)
def test_logprobs_grad_of_some_rows(dev):
    """The statistics of a batch, cut like its logits: a gradient by parts."""
    z, tok = logits(9, 700, torch.bfloat16, seed=39)
    z, tok, g = z.to(dev), tok.to(dev), torch.randn(9, generator=gen(40)).to(dev)
    r = token_logprobs(z, tok, temperature=1.5)
    whole = token_logprobs_grad(z, tok, r, g, g)
    for lo, hi in ((0, 4), (4, 9), (3, 4)):
        part = dataclasses.replace(r, stat=r.stat[:, lo:hi])
        assert torch.equal(token_logprobs_grad(z[lo:hi], tok[lo:hi], part, g[lo:hi], g[lo:hi]), whole[lo:hi])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [1e-12, 1e12])
def test_logprobs_grad_temperatures(dev, T):
    """Temperatures that leave the largest logit alone, or all of them alike."""
    z, tok = logits(6, 700, torch.float32, seed=26)
    z[1, 5:] = -math.inf
    z[2, :300] = torch.finfo(torch.float32).min
    z[3] = 0.25
    tok[1] = 2
    check_token_grad(z, tok, None, torch.randn(6, generator=gen(27)), T, dev)
    check_token_grad(z, tok, torch.randn(6, generator=gen(28)), torch.randn(6, generator=gen(29)), T, dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_logprobs_grad_against_differences(dev):
    """(f(z + s d) - f(z - s d)) / 2 s is off by the roundings of f (each below SUM (1 + ln V), n of them) over s and
    by s^2 / 6 of the third derivative, which for these functions and |d| <= 1 stays below 12 n."""
    n, V, T, s = 4, 37, 1.3, 2.0 ** -5
    z, tok = logits(n, V, torch.float32, seed=8)
    z, tok = z.to(dev), tok.to(dev)
    g, h = torch.rand(n, generator=gen(9)).to(dev), torch.rand(n, generator=gen(10)).to(dev)
    d = (torch.rand(n, V, generator=gen(11)) * 2 - 1).to(dev)

    def f(x):
        r = token_logprobs(x, tok, temperature=T)
        return (g * r.logprob + h * r.entropy).double().sum().item()

    got = (token_logprobs_grad(z, tok, token_logprobs(z, tok, temperature=T), g, h).double() * d.double()).sum().item()
    assert abs(got - (f(z + s * d) - f(z - s * d)) / (2 * s)) <= 2 * n * SUM * (1 + math.log(V)) / s + 2 * n * s * s


# ---- distillation ---------------------------------------------------------------------------------------------------

def teacher_of(rows, V, dtype=torch.float32):
    """rows: lists of (column, value)."""
    ptr = torch.tensor([0] + [len(r) for r in rows]).cumsum(0)
    flat = [e for r in rows for e in r]
    return CSR(len(rows), V, ptr, torch.tensor([c for c, _ in flat], dtype=torch.int32),
               torch.tensor([v for _, v in flat], dtype=torch.float32).to(dtype))


def random_teacher(n, V, most, seed, dtype=torch.float32):
    g = gen(seed)
    rows = []
    for _ in range(n):
        k = int(torch.randint(0, most + 1, (1,), generator=g))
        rows.append([(int(c), float(v)) for c, v in zip(torch.randperm(V, generator=g)[:k], torch.randn(k, generator=g) * 2)])
    return teacher_of(rows, V, dtype)


def ref_distill(z, T, tau, w):
    n, V = z.shape
    logq, q, _ = ref_logprobs(z, tau)
    loss = torch.zeros(n, dtype=torch.float64)
    grad = torch.zeros(n, V, dtype=torch.float64)
    most = torch.zeros(n, dtype=torch.float64)
    mag = torch.zeros(n, V, dtype=torch.float64)
    ptr = T.rowptr.cpu().tolist()
    for i in range(n):
        c, v = T.col.cpu()[ptr[i]:ptr[i + 1]].long(), T.val.cpu()[ptr[i]:ptr[i + 1]].double()
        c, v = c[c != -1], v[c != -1]
        if ((c < 0) | (c >= V)).any() or v.isnan().any() or (v == math.inf).any():
            loss[i], grad[i] = math.nan, (0.0 if w[i] == 0 else math.nan)
            continue
        if c.numel() == 0 or (v == -math.inf).all():
            continue
        logp = torch.log_softmax(v / tau, 0)
        p = logp.exp()
        term = torch.where(p == 0, 0.0, p * (logp - logq[i, c]))
        loss[i] = term.sum()
        most[i] = torch.where(p == 0, 0.0, p * (logp.abs() + logq[i, c].abs())).sum().nan_to_num(0, posinf=0)
        if w[i] != 0:
            dense = torch.zeros(V, dtype=torch.float64).index_add(0, c, p)
            grad[i] = w[i] * (q[i] - dense) / tau
            mag[i] = w[i].abs() * (q[i] + dense) / tau
    return loss, most, grad, mag


def check_distill(z, T, tau, w, dev, inplace=False):
    n, V = z.shape
    loss, most, grad, mag = ref_distill(z, T, tau, torch.ones(n).double() if w is None else w.double())
    tol = SUM * (1 + most + math.log(V))
    zd, Td, wd = z.clone().to(dev), T.to(dev), None if w is None else w.to(dev)
    a = distill_loss(zd, Td, temperature=tau)
    near(a.loss, loss, tol)
    gtol = half_step(z.dtype, grad) + 2 * SUM * mag.nan_to_num(0.0)
    near(distill_grad(zd, Td, a, weight=wd), grad, gtol)
    b, dz = distill_loss_grad(zd, Td, weight=wd, temperature=tau, out=zd if inplace else None)
    near(b.loss, loss, tol)
    near(dz, grad, gtol)
    if inplace:
        assert dz is zd
    return dz


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,most", [(1, 1, 1), (5, 7, 7), (4, 100, 20), (3, 2049, 64), (3, 4100, 70), (2, 8200, 300),
                                      (3, 16389, 100), (2, 40001, 33)])
def test_distill(dev, dtype, n, V, most):
    z, _ = logits(n, V, dtype, seed=12)
    w = torch.rand(n, generator=gen(13)) + 0.1
    check_distill(z, random_teacher(n, V, most, seed=V), 1.0, None, dev)
    check_distill(z, random_teacher(n, V, most, seed=V + 1, dtype=torch.bfloat16), 2.0, w, dev)
    check_distill(z, random_teacher(n, V, most, seed=V + 2, dtype=torch.float16), 0.8, w, dev, inplace=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V", [(300, 1000), (700, 2049), (530, 5001), (300, 20003), (2500, 300)])
def test_distill_many_rows(dtype, n, V):
    z, _ = logits(n, V, dtype, seed=14)
    w = torch.rand(n, generator=gen(15))
    w[3] = 0.0
    T = random_teacher(n, V, 40, seed=V)
    check_distill(z, T, 1.5, w, "cuda")
    check_distill(z, T, 1.0, w, "cuda", inplace=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_many_long_rows(dtype):
    """More workgroups than are on the chip at once, rows longer than one of them holds."""
    z, _ = logits(130, 131100, dtype, seed=41)
    w = torch.rand(130, generator=gen(42)) + 0.1
    w[5] = 0.0
    check_distill(z, random_teacher(130, 131100, 90, seed=43), 1.5, w, "cuda", inplace=True)


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_long_teacher_rows(dev):
    """Thousands of entries a row: ascending columns, absent ones behind them, one column twice, any order."""
    V, L = 9000, 3001
    z, _ = logits(5, V, torch.float32, seed=30)
    g = gen(31)
    rows = []
    for i in range(5):
        c = torch.randperm(V, generator=g)[:L]
        c = c if i == 4 else c.sort().values
        if i == 1:
            c[2000:] = -1
        if i == 2:
            c[1500] = c[1499]
        if i == 3:
            c[10] = -1                                     # absent in the middle
        rows.append([(int(x), float(v)) for x, v in zip(c, torch.randn(L, generator=g) * 2)])
    w = torch.rand(5, generator=gen(32)) + 0.1
    for dtype in (torch.float32, torch.bfloat16):
        check_distill(z.to(dtype), teacher_of(rows, V), 1.5, w, dev, inplace=True)


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_rows(dev):
    V = 3000
    z, _ = logits(16, V, torch.float32, seed=16)
    inf = math.inf
    rows = [[],                                             # no entry
            [(5, -inf), (6, -inf)],                         # no mass
            [(7, 1.0)],                                     # all mass on one
            [(7, 1.0), (9, 2.0), (7, 1.0), (9, 0.5)],       # columns twice
            [(-1, 3.0), (4, 1.0), (-1, 9.0)],               # padded to a length
            [(-1, 0.0)],
            [(0, 1.0), (V, 2.0)],                           # outside the vocabulary
            [(0, 1.0), (-2, 2.0)],
            [(2, 0.5), (3, -inf), (4, 1.5)],
            [(0, 0.0), (V - 1, 0.0)],
            [(1, 1.0), (2, 1.0)],                           # the student masks one of them
            [(1, 1.0), (2, 1.0)],                           # the student masks everything
            [(11, 2.0), (12, 1.0)],
            [(11, 2.0), (12, math.nan)],
            [(11, inf), (12, 0.0)],
            [(j * 2, float(j % 7)) for j in range(1400)]]   # more entries than are staged at once
    z[10, 2] = -inf
    z[11] = -inf
    z[0] = math.nan                                          # garbage in a row that is not trained on
    z[12, 5:11] = -inf
    w = torch.linspace(0.5, 2.0, 16)
    w[12] = 0.0
    dz = check_distill(z, teacher_of(rows, V), 1.2, w, dev)
    assert (dz[0] == 0).all() and (dz[12] == 0).all()
    many = torch.randn(2, V, generator=gen(17))
    twice = [[(j % 900, float(j % 5)) for j in range(2500)], [(5, 1.0)] * 2048]
    check_distill(many, teacher_of(twice, V), 1.0, None, dev, inplace=True)


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_layouts(dev):
    V = 501
    z, _ = logits(6, V, torch.bfloat16, seed=18)
    T = random_teacher(6, V, 20, seed=19)
    wide = torch.zeros(6, 700, dtype=torch.bfloat16, device=dev)
    wide[:, 99:600] = z.to(dev)
    a, da = distill_loss_grad(z.to(dev), T.to(dev))
    out = torch.full((6, 600), 3.0, dtype=torch.bfloat16, device=dev)
    b, db = distill_loss_grad(wide[:, 99:600], T.to(dev), out=out[:, 50:551])
    assert torch.equal(a.loss, b.loss) and torch.equal(da, db)
    assert (out[:, :50] == 3).all() and (out[:, 551:] == 3).all()
    one = torch.full((1,), 0.25, device=dev).expand(6)       # one weight for all rows
    check = distill_loss_grad(z.to(dev), T.to(dev), weight=one)[1]
    assert torch.equal(check, distill_loss_grad(z.to(dev), T.to(dev), weight=one.contiguous())[1])
    e = CSR(0, V, torch.zeros(1, dtype=torch.int64, device=dev), T.col[:0].to(dev), T.val[:0].to(dev))
    r, dz = distill_loss_grad(z[:0].to(dev), e)
    assert r.loss.shape == (0,) and dz.shape == (0, V)
    # a row pointer that leaves the arrays stays inside them
    bad = CSR(6, V, torch.tensor([0, 10 ** 9, -5, 3, 2, 10 ** 12, 7], device=dev), T.col.to(dev), T.val.to(dev))
    assert distill_loss(z.to(dev), bad).loss.shape == (6,)


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_against_differences(dev):
    """As for the log-probabilities: n losses, each off by SUM (1 + its terms); third derivative of ln Z below 2 n / tau^3."""
    n, V, tau, s = 5, 41, 1.4, 2.0 ** -5
    z, _ = logits(n, V, torch.float32, seed=20)
    z, T = z.to(dev), random_teacher(n, V, 9, seed=21).to(dev)
    w = torch.rand(n, generator=gen(22)).to(dev)
    d = (torch.rand(n, V, generator=gen(23)) * 2 - 1).to(dev)
    f = lambda x: (w * distill_loss(x, T, temperature=tau).loss).double().sum().item()  # noqa: E731
    got = (distill_loss_grad(z, T, weight=w, temperature=tau)[1].double() * d.double()).sum().item()
    assert abs(got - (f(z + s * d) - f(z - s * d)) / (2 * s)) <= n * SUM * (1 + 12) / s + n * s * s


# ---- together -------------------------------------------------------------------------------------------------------

def train(dev, dtype):
    """One distillation step of a tied lookup-and-project model from a teacher's alternatives."""
    g = gen(30)
    V, D, n, k, tau = 300, 64, 50, 12, 2.0
    W = (torch.randn(V, D, generator=g) / 8).to(dtype).to(dev)
    tok = torch.randint(0, V, (n,), generator=g).to(dev)
    tok[7] = -1
    big = (torch.randn(n, V, generator=g) * 2).to(dtype).to(dev)
    top = token_logprobs(big, tok, k=k).top
    H = embedding(W, tok, scale=8.0)
    Z = (H.float() @ W.float().t()).to(dtype)
    w = torch.full((n,), 1.0 / n, device=dev)
    w[7] = 0.0
    loss, dZ = distill_loss_grad(Z, top, weight=w, temperature=tau)
    dH = (dZ.float() @ W.float()).to(dtype)
    dW = dZ.float().t() @ H.float()
    embedding_grad(dH, tok, V, scale=8.0, dtype=torch.float32, out=dW, accumulate=True)
    return W, tok, big, top, w, tau, loss.loss, dW


@pytest.mark.parametrize("dev", DEVICES)
def test_step_of_a_tied_model(dev):
    W, tok, big, top, w, tau, loss, dW = train(dev, torch.float32)
    W, tok, big, w = W.cpu().double().requires_grad_(), tok.cpu(), big.cpu().double(), w.cpu().double()
    T = torch.full_like(big, -math.inf)
    idx = order_of(big, 12)
    T.scatter_(1, idx, torch.log_softmax(big, 1).gather(1, idx))
    p = torch.softmax(T / tau, 1)
    H = torch.where(tok[:, None] >= 0, W[tok.clamp_min(0)] * 8.0, 0.0)
    logq = torch.log_softmax(H @ W.t() / tau, 1)
    ref = (torch.xlogy(p, p) - p * logq).sum(1)
    (ref * w).sum().backward()
    near(loss, ref.detach(), torch.tensor(1e-4))
    # 50 tokens of weight 1/50 through products of 64 and 300 terms: each below 400 roundings of terms below 8
    near(dW, W.grad, torch.tensor(8 * SUM))


def decode(dev, dtype):
    g = gen(31)
    V, D = 1000, 128
    W = (torch.randn(V, D, generator=g) / 11).to(dtype).to(dev)
    tok = torch.tensor([5, 999, 0, 17], device=dev)
    seen = []
    for _ in range(3):   # one token of each sequence at a time, the likeliest next
        z = (embedding(W, tok, scale=11.0).float() @ W.float().t()).to(dtype)
        z.scatter_(1, tok[:, None], -math.inf)     # no token twice in a row
        r = token_logprobs(z, tok, k=5, temperature=0.8)
        assert (r.logprob == -math.inf).all()
        tok = r.top.col.view(4, 5)[:, 0].long()
        seen.append((tok.clone(), r.top.val.view(4, 5)[:, 0].clone()))
    return seen


@pytest.mark.gpu
def test_decode_like_the_cpu():
    for (a, x), (b, y) in zip(decode("cuda", torch.float32), decode("cpu", torch.float32)):
        assert torch.equal(a.cpu(), b)
        near(x, y, torch.tensor(1e-4))


# ---- streams, graphs, sizes past 32 bits ----------------------------------------------------------------------------

@pytest.mark.gpu
def test_captured_and_replayed():
    """All calls of a step in two HIP graphs whose replays alternate with eager work on changing inputs."""
    dev = torch.device("cuda")
    V, D, n, k = 5000, 96, 300, 7
    W = torch.randn(V, D, device=dev).bfloat16()
    z = torch.randn(n, V, device=dev).bfloat16()
    tok = torch.randint(0, V, (n,), device=dev)
    g = torch.rand(n, device=dev)

    def step():
        y = embedding(W, tok, scale=3.0)
        r = token_logprobs(z, tok, k=k)
        dz = token_logprobs_grad(z, tok, r, g_logprob=g, g_entropy=g)
        d, dd = distill_loss_grad(z, r.top, weight=g, temperature=2.0)
        dw = embedding_grad(y, tok, V)
        return [y, r.logprob, r.entropy, r.top.col, r.top.val, dz, d.loss, dd, dw]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step()
        graphs.append((gr, outs))
    for i in range(4):
        z.copy_(torch.randn(n, V, device=dev).bfloat16())
        tok.copy_(torch.randint(-1, V, (n,), device=dev))
        for gr, _ in graphs:
            gr.replay()
        for a, b, c in zip(step(), graphs[0][1], graphs[1][1]):
            assert torch.equal(a, b) and torch.equal(a, c)
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 1500, 13000])
def test_captured_gradients(n):
    """Every way of the table's gradient in a graph: unsorted, sorted in one launch, in several."""
    dev, V, D = torch.device("cuda"), 4001, 72
    dY, tok = torch.randn(n, D, device=dev).bfloat16(), torch.randint(0, V, (n,), device=dev)
    main = torch.zeros(V, D, device=dev)
    embedding_grad(dY, tok, V)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        dW = embedding_grad(dY, tok, V)
        embedding_grad(dY, tok, V, out=main, accumulate=True)
    total = torch.zeros(V, D, device=dev)
    for i in range(4):
        dY.copy_(torch.randn(n, D, device=dev).bfloat16())
        tok.copy_(torch.randint(-1, V, (n,), device=dev))
        gr.replay()
        assert torch.equal(dW, embedding_grad(dY, tok, V))
        embedding_grad(dY, tok, V, out=total, accumulate=True)
        assert torch.equal(main, total)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_on_another_stream():
    dev = torch.device("cuda")
    W, tok = torch.randn(3000, 200, device=dev), torch.randint(0, 3000, (9000,), device=dev)
    z = torch.randn(64, 3000, device=dev)
    want = [embedding_grad(embedding(W, tok), tok, 3000), token_logprobs(z, tok[:64], k=20).top.val]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:     # two calls in flight at once, each with its own workspace
        with torch.cuda.stream(s):
            got.append([embedding_grad(embedding(W, tok), tok, 3000), token_logprobs(z, tok[:64], k=20).top.val])
    torch.cuda.synchronize()
    for r in got:
        assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])


@pytest.mark.gpu
def test_rows_past_32_bits():
    """Offsets beyond 2^31 elements: the last rows are those of a small call."""
    dev = torch.device("cuda")
    n, V = 17000, 131072
    z = torch.empty(n, V, dtype=torch.bfloat16, device=dev)
    z[-40:] = torch.randn(40, V, device=dev)
    z[:-40] = z[-40]
    tok = torch.randint(0, V, (n,), device=dev)
    a, b = token_logprobs(z, tok, k=3), token_logprobs(z[-40:].clone(), tok[-40:], k=3)
    assert torch.equal(a.logprob[-40:], b.logprob) and torch.equal(a.top.col.view(n, 3)[-40:], b.top.col.view(40, 3))
    g = torch.rand(n, device=dev)
    want = token_logprobs_grad(z[-40:].clone(), tok[-40:], b, g[-40:])
    dd = distill_loss_grad(z[-40:].clone(), b.top, weight=g[-40:])[1]
    T = CSR(n, V, a.top.rowptr, a.top.col, a.top.val)
    assert torch.equal(distill_loss_grad(z, T, weight=g)[1][-40:], dd)
    assert torch.equal(token_logprobs_grad(z, tok, a, g, out=z)[-40:], want)
    del z, T, a
    V, D = 600_000, 4096
    W = torch.empty(V, D, dtype=torch.bfloat16, device=dev)
    W[-5:] = torch.randn(5, D, device=dev)
    tok = torch.tensor([V - 1, V - 5, 3, V - 1], device=dev)
    W[3] = 1.0
    y = embedding(W, tok)
    assert torch.equal(y, W[tok])
    dw = embedding_grad(y, tok, V, out=W)
    assert torch.equal(dw[-1].float(), 2 * y[0].float()) and torch.equal(dw[-5], y[1]) and torch.equal(dw[3], y[2])
    assert (dw[-4:-1] == 0).all() and (dw[4:100] == 0).all()


# ---- refusals -------------------------------------------------------------------------------------------------------

def refused(call, text):
    with pytest.raises(ValueError, match=text):
        call()


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals_embedding(dev):
    W, tok, dY = torch.randn(9, 4, device=dev), torch.tensor([1, 2], device=dev), torch.randn(2, 4, device=dev)
    refused(lambda: embedding(W[0], tok), "2 dimensions")
    refused(lambda: embedding(W.double(), tok), "float32, bfloat16 or float16")
    refused(lambda: embedding(W, tok.float()), "int32 or int64")
    refused(lambda: embedding(W, tok, scale=math.inf), "finite")
    refused(lambda: embedding(W, tok, out=W[:3]), "must be")
    refused(lambda: embedding(W, tok, out=W[2:4]), "overlaps")
    refused(lambda: embedding(W, tok, out=torch.empty(2, 4, device=dev).bfloat16()), "must be")
    refused(lambda: embedding(W, tok, out=torch.empty(4, 2, device=dev).t()), "adjacent")
    refused(lambda: embedding(W, tok, out=torch.empty(4, device=dev).expand(2, 4)), "overlap")
    refused(lambda: embedding(W.requires_grad_(), tok), "autograd")
    with torch.no_grad():
        embedding(W, tok)
    refused(lambda: embedding_grad(dY, tok, 0), "positive")
    refused(lambda: embedding_grad(dY[:1], tok, 9), "dY must be")
    refused(lambda: embedding_grad(dY, tok, 9, accumulate=True), "accumulate")
    refused(lambda: embedding_grad(dY, tok, 9, dtype=torch.bfloat16), "dtype")
    refused(lambda: embedding_grad(dY.bfloat16(), tok, 9, out=torch.empty(9, 4, device=dev), dtype=torch.bfloat16), "must be")
    refused(lambda: embedding_grad(dY, tok, 9, out=torch.empty(8, 4, device=dev)), "must be")
    buf = torch.empty(20, 4, device=dev)
    refused(lambda: embedding_grad(buf[8:10], tok, 9, out=buf[:9]), "overlaps")


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals_logits(dev):
    z, tok = torch.randn(3, 10, device=dev), torch.tensor([1, 2, 3], device=dev)
    r = token_logprobs(z, tok, k=2)
    refused(lambda: token_logprobs(z[0], tok), "2 dimensions")
    refused(lambda: token_logprobs(z.double(), tok), "float32, bfloat16 or float16")
    refused(lambda: token_logprobs(z[:, :0], tok), "vocabulary")
    refused(lambda: token_logprobs(z, tok[:2]), "tokens must be")
    refused(lambda: token_logprobs(z, tok, k=11), "between 0 and 10")
    refused(lambda: token_logprobs(torch.zeros(3, 500, device=dev), tok, k=129), "between 0 and 128")
    for t in (0.0, -1.0, math.nan, math.inf):
        refused(lambda: token_logprobs(z, tok, temperature=t), "temperature")
    refused(lambda: token_logprobs_grad(z[:2], tok[:2], r), "stats are of")
    refused(lambda: token_logprobs_grad(z, tok, r, g_logprob=torch.ones(2, device=dev)), "g_logprob must be")
    refused(lambda: token_logprobs_grad(z, tok, r, g_entropy=tok), "floating")
    refused(lambda: token_logprobs_grad(z, tok, r, out=torch.empty(3, 10, device=dev).half()), "must be")
    buf = torch.randn(5, 10, device=dev)
    refused(lambda: token_logprobs_grad(buf[:3], tok, r, out=buf[1:4]), "overlaps")
    refused(lambda: token_logprobs(z.clone().requires_grad_(), tok), "autograd")
    T = r.top
    refused(lambda: distill_loss(z[:2], T), "teacher is")
    refused(lambda: distill_loss(z, CSR(3, 10, T.rowptr.int(), T.col, T.val)), "rowptr")
    refused(lambda: distill_loss(z, CSR(3, 10, T.rowptr[:3], T.col, T.val)), "rowptr")
    refused(lambda: distill_loss(z, CSR(3, 10, T.rowptr, T.col.long(), T.val)), "col")
    refused(lambda: distill_loss(z, CSR(3, 10, T.rowptr, T.col, T.val[:3])), "val")
    refused(lambda: distill_loss(z, CSR(3, 10, T.rowptr, T.col, T.val.double())), "val")
    refused(lambda: distill_loss(z, T, temperature=0), "temperature")
    refused(lambda: distill_loss_grad(z, T, weight=torch.ones(4, device=dev)), "weight must be")
    refused(lambda: distill_loss_grad(buf[:3], T, out=buf[2:5]), "overlaps")
    s = distill_loss(z, T)
    refused(lambda: distill_grad(z, CSR(3, 10, T.rowptr, T.col[:5], T.val[:5]), s), "stats are of")
    if dev == "cuda":
        refused(lambda: distill_loss(z, T.to("cpu")), "is on")
        refused(lambda: token_logprobs(z, tok.cpu()), "is on")


# ---- distillation: rows that fill a CU's registers, teacher rows against a large vocabulary --------------------------

def teacher_with_equal_columns(n, V, least, most, seed):
    """Rows of `least` to `most` entries in any order, with columns twice in a
    row's first 64 entries and further apart, one of them three times, and
    absent entries."""
    g = gen(seed)
    rows = []
    for i in range(n):
        L = least + int(torch.randint(0, most - least + 1, (1,), generator=g))
        c = torch.randperm(V, generator=g)[:L]
        c[L - 1] = c[3]
        c[7] = c[3]
        c[L // 2] = c[L - 2]
        c[20] = c[21]
        c[30] = c[L - 4] = -1
        c[0], c[L - 3] = 0, V - 1                            # beside the row's vectors
        rows.append([(int(x), float(v)) for x, v in zip(c, torch.randn(L, generator=g) * 2)])
    return teacher_of(rows, V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V", [(260, 40001), (256, 65532), (257, 33024)])
def test_distill_rows_that_fill_a_cu(dtype, n, V):
    """16-bit rows of 17 to 32 pages, many of them: a workgroup of 1024 threads holds one."""
    z, _ = logits(n, V, dtype, seed=50)
    z[5, 17:9000] = -math.inf
    w = torch.rand(n, generator=gen(51)) + 0.1
    w[3] = 0.0
    check_distill(z, random_teacher(n, V, 90, seed=V), 1.5, w, "cuda")
    check_distill(z, teacher_with_equal_columns(n, V, 66, 200, seed=52), 1.0, w, "cuda", inplace=True)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_equal_columns_in_a_large_vocabulary(dev, dtype):
    """65 to 128 entries against 300001 columns: equal ones are found by a search among all entries."""
    z, _ = logits(3, 300001, dtype, seed=53)
    w = torch.tensor([0.5, 1.25, 2.0])
    for seed in (54, 55):
        T = teacher_with_equal_columns(3, 300001, 65, 128, seed=seed)
        check_distill(z, T, 1.3, w, dev)
        check_distill(z, T, 1.0, None, dev, inplace=True)


@pytest.mark.gpu
def test_distill_equal_columns_of_many_rows_in_a_large_vocabulary():
    """The same where a launch of its own ends the rows."""
    z, _ = logits(40, 300001, torch.float32, seed=56)
    w = torch.rand(40, generator=gen(57)) + 0.1
    check_distill(z, teacher_with_equal_columns(40, 300001, 65, 128, seed=58), 1.3, w, "cuda", inplace=True)
