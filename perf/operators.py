"""Operators of rows over a vocabulary: embedding lookup and gradient, token log-probabilities, distillation.

Each case is one pass as a program makes it.  ``own`` false: plain torch operations in 32 bits; ``own`` true: the
framework's operators (``spmm_amd.ops.embedding``, ``.logprobs``, ``.distill``).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the input of one decode step: one token for each of 32 running sequences
        dict(name="lookup decode", op="lookup", n=32, v=65536, d=2048, dtype="bf16", pad=0.0),
        # the input of a packed training batch
        dict(name="lookup batch", op="lookup", n=32768, v=131072, d=4096, dtype="bf16", pad=0.0),
        # full precision, a width that is no multiple of anything, a fifth of the batch is padding
        dict(name="lookup padded odd", op="lookup", n=5001, v=50021, d=1111, dtype="fp32", pad=0.2),
        # the dense gradient of a training batch: most rows of the table get no token
        dict(name="grad batch", op="grad", n=16384, v=131072, d=4096, dtype="bf16", to="bf16", add=False, pad=0.0),
        # micro-batches accumulate into a 32-bit main gradient
        dict(name="grad accumulate", op="grad", n=65536, v=65536, d=1024, dtype="bf16", to="fp32", add=True, pad=0.0),
        # a short fine-tuning batch with padding in half precision
        dict(name="grad short", op="grad", n=777, v=32003, d=1000, dtype="fp16", to="fp16", add=False, pad=0.1),
        # one decode step of 8 sequences under a grammar's mask, 20 alternatives each, sampled at 0.7
        dict(name="logprobs decode", op="logprobs", n=8, v=131072, dtype="bf16", k=20, temp=0.7, masked=0.3),
        # a prompt's tokens scored, 5 alternatives each, a vocabulary of odd size
        dict(name="logprobs prompt", op="logprobs", n=4096, v=100003, dtype="bf16", k=5, temp=1.0, masked=0.0),
        # a policy's update: log-probabilities and entropies, then their gradient
        dict(name="logprobs train", op="policy", n=2048, v=65536, dtype="fp32", temp=1.0),
        # a training step's loss and gradient from 64 teacher logits a token
        dict(name="distill train", op="distill", n=4096, v=131072, dtype="bf16", k=64, ragged=False, temp=2.0, grad=True),
        # held-out loss against teacher rows cut to their nucleus: from none to 100 entries
        dict(name="distill evaluate", op="distill", n=1500, v=50021, dtype="fp32", k=100, ragged=True, temp=1.0, grad=False),
        # a small student's short batch
        dict(name="distill short", op="distill", n=48, v=32768, dtype="fp16", k=32, ragged=True, temp=1.5, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "logprobs", "policy", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    odd = rng.random() < 0.5
    if op in ("lookup", "grad"):
        v, d = _log(rng, 1000, 131072), _log(rng, 64, 4096)
        if not odd:
            v, d = max(8, v // 8 * 8), max(8, d // 8 * 8)
        n = _log(rng, 1, 32768)
        pad = rng.choice([0.0, 0.1, 0.5])
        if op == "lookup":
            return dict(op=op, n=n, v=v, d=d, dtype=dtype, pad=pad)
        return dict(op=op, n=n, v=v, d=d, dtype=dtype, to=rng.choice([dtype, "fp32"]), add=rng.random() < 0.4, pad=pad)
    v = _log(rng, 1000, 131072)
    if not odd:
        v = max(8, v // 8 * 8)
    n = _log(rng, 1, max(1, min(8192, (1 << 27) // v)))
    temp = rng.choice([0.7, 1.0, 1.0, 2.0])
    if op == "logprobs":
        return dict(op=op, n=n, v=v, dtype=dtype, k=rng.choice([0, 1, 5, 20, 64, 100]), temp=temp, masked=rng.choice([0.0, 0.0, 0.3, 0.95]))
    if op == "policy":
        return dict(op=op, n=n, v=v, dtype=dtype, temp=temp)
    return dict(op=op, n=n, v=v, dtype=dtype, k=_log(rng, 1, 256), ragged=rng.random() < 0.5, temp=temp, grad=rng.random() < 0.7)


def _tokens(case, g):
    """Word frequencies fall as 1 / rank; which token has which rank is random."""
    n, v = case["n"], case["v"]
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(v + 1)).floor().long() - 1
    tok = torch.randperm(v, generator=g, device="cuda")[rank.clamp_(0, v - 1)]
    if case["pad"]:
        tok[1:][torch.rand(n - 1, generator=g, device="cuda") < case["pad"]] = -1
    return tok


def _logits(n, v, g):
    """Bell-shaped logits with a few likely tokens in each row."""
    z = torch.randn(n, v, generator=g, device="cuda") * 2.5
    peak = torch.randint(0, v, (n, 8), generator=g, device="cuda")
    return z.scatter_(1, peak, 6 + 6 * torch.rand(n, 8, generator=g, device="cuda"))


def _loss_scale(case):
    """Half-precision gradients are kept in range by a scaled loss."""
    return 1024.0 if case["dtype"] == "fp16" else 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    n, v, op = case["n"], case["v"], case["op"]
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if op in ("lookup", "grad"):
        d = case["d"]
        s["tokens"] = _tokens(case, g)
        s["scale"] = math.sqrt(d)
        if op == "lookup":
            s["w"] = (torch.randn(v, d, generator=g, device="cuda") / math.sqrt(d)).to(dt)
            return s
        s["dy"] = (torch.randn(n, d, generator=g, device="cuda") * 0.01).to(dt)
        if case["add"]:   # what earlier micro-batches left
            s["dw"] = (torch.randn(v, d, generator=g, device="cuda") * 0.1).to(DTYPES[case["to"]])
        return s
    z = _logits(n, v, g)
    if op == "logprobs" and case["masked"]:   # a grammar forbids tokens; every row keeps some
        z.masked_fill_(torch.rand(v, generator=g, device="cuda")[None, :] < case["masked"], -math.inf)
        z[:, :: max(1, v // 64)] = z[:, :: max(1, v // 64)].clamp_min(-4.0)
    s["logits"] = z.to(dt)
    if op in ("logprobs", "policy"):
        noise = -torch.log(-torch.log(torch.rand(n, v, generator=g, device="cuda").clamp_(1e-20, 1 - 1e-7)))
        s["tokens"] = (z / case["temp"] + noise).argmax(1)   # sampled from the row itself
        if op == "policy":
            s["g_logprob"] = torch.randn(n, generator=g, device="cuda") * _loss_scale(case) / n
            s["g_entropy"] = torch.full((n,), -0.01 * _loss_scale(case) / n, device="cuda")
        return s
    k = min(case["k"], v)
    teacher = z * 0.9 + torch.randn(n, v, generator=g, device="cuda")
    val, col = teacher.topk(k, dim=1)
    count = torch.randint(0, k + 1, (n,), generator=g, device="cuda") if case["ragged"] else torch.full((n,), k, device="cuda")
    count[0] = k
    keep = torch.arange(k, device="cuda")[None, :] < count[:, None]
    s["rowptr"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), count.cumsum(0)])
    s["col"], s["val"] = col[keep].to(torch.int32), val[keep].float()
    if case["grad"]:
        s["weight"] = torch.full((n,), _loss_scale(case) / n, device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _softmax_parts(z, temp):
    """(t, log of the sum of exp t) with t = (z - row maximum) / temp."""
    t = (z - z.amax(1, keepdim=True)) / temp
    return t, t.exp().sum(1).log()


def _plain_lookup(s):
    w, tok = s["w"], s["tokens"]
    rows = w[tok.clamp_min(0)].float() * s["scale"]
    return torch.where(tok[:, None] >= 0, rows, 0.0).to(w.dtype)


def _plain_grad(s):
    case, tok, dy = s["case"], s["tokens"], s["dy"]
    at = torch.where(tok < 0, case["v"], tok)   # padding goes to a row that is dropped
    acc = torch.zeros(case["v"] + 1, case["d"], device=dy.device).index_add_(0, at, dy.float())[: case["v"]] * s["scale"]
    if not case["add"]:
        return acc.to(DTYPES[case["to"]])
    return s["dw"].copy_((s["dw"].float() + acc).to(s["dw"].dtype))


def _plain_logprobs(s, alternatives):
    z, case = s["logits"].float(), s["case"]
    t, logz = _softmax_parts(z, case["temp"])
    logprob = t.gather(1, s["tokens"][:, None])[:, 0] - logz
    q = (t - logz[:, None]).exp()
    entropy = logz - torch.where(q > 0, q * t, 0.0).sum(1)
    if not alternatives:
        return logprob, entropy, q, t - logz[:, None]
    if not case["k"]:
        return logprob, entropy
    # larger logits first, the lower index first among equal ones: one whole number holds both
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits)
    v = z.shape[1]
    key = order * (1 << 20) + (v - 1 - torch.arange(v, device=z.device))[None, :]
    index = v - 1 - (key.topk(min(case["k"], v), dim=1).values & ((1 << 20) - 1))
    return logprob, entropy, index.to(torch.int32), t.gather(1, index) - logz[:, None]


def _plain_policy(s):
    logprob, entropy, q, logq = _plain_logprobs(s, False)
    g, h, temp = s["g_logprob"][:, None], s["g_entropy"][:, None], s["case"]["temp"]
    dz = -g * q - h * torch.where(q > 0, q * (logq + entropy[:, None]), 0.0)
    dz.scatter_add_(1, s["tokens"][:, None], g)
    return logprob, entropy, (dz / temp).to(s["logits"].dtype)


def _plain_distill(s):
    case, rowptr, col = s["case"], s["rowptr"], s["col"].long()
    z, temp, n = s["logits"].float(), case["temp"], case["n"]
    count = rowptr[1:] - rowptr[:-1]
    row = torch.repeat_interleave(torch.arange(n, device=z.device), count, output_size=col.numel())
    u = s["val"] / temp
    u = u - torch.full((n,), -math.inf, device=z.device).scatter_reduce_(0, row, u, "amax")[row]
    p = u.exp()
    total = torch.zeros(n, device=z.device).index_add_(0, row, p)[row]
    p, logp = p / total, u - total.log()
    t, logz = _softmax_parts(z, temp)
    loss = torch.zeros(n, device=z.device).index_add_(0, row, p * (logp - t[row, col] + logz[row]))
    if not case["grad"]:
        return loss
    weight = torch.where(count > 0, s["weight"], 0.0)
    dz = (t - logz[:, None]).exp()
    dz.index_put_((row, col), -p, accumulate=True)
    return loss, (dz * (weight / temp)[:, None]).to(s["logits"].dtype)


# ---- the framework's operators --------------------------------------------------------------------------------------

def _own(s):
    from spmm_amd.ops.csr import CSR
    from spmm_amd.ops.distill import distill_loss, distill_loss_grad
    from spmm_amd.ops.embedding import embedding, embedding_grad
    from spmm_amd.ops.logprobs import token_logprobs, token_logprobs_grad

    case, op = s["case"], s["case"]["op"]
    if op == "lookup":
        return embedding(s["w"], s["tokens"], scale=s["scale"])
    if op == "grad":
        return embedding_grad(s["dy"], s["tokens"], case["v"], scale=s["scale"], dtype=DTYPES[case["to"]],
                              out=s.get("dw"), accumulate=case["add"])
    if op == "logprobs":
        r = token_logprobs(s["logits"], s["tokens"], k=min(case["k"], case["v"]), temperature=case["temp"])
        if not case["k"]:
            return r.logprob, r.entropy
        return r.logprob, r.entropy, r.top.col.view(case["n"], -1), r.top.val.view(case["n"], -1)
    if op == "policy":
        r = token_logprobs(s["logits"], s["tokens"], temperature=case["temp"])
        dz = token_logprobs_grad(s["logits"], s["tokens"], r, g_logprob=s["g_logprob"], g_entropy=s["g_entropy"])
        return r.logprob, r.entropy, dz
    teacher = CSR(case["n"], case["v"], s["rowptr"], s["col"], s["val"])
    if not case["grad"]:
        return distill_loss(s["logits"], teacher, temperature=case["temp"]).loss
    r, dz = distill_loss_grad(s["logits"], teacher, weight=s["weight"], temperature=case["temp"])
    return r.loss, dz


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "lookup":
        return _plain_lookup(state)
    if op == "grad":
        return _plain_grad(state)
    if op == "logprobs":
        return _plain_logprobs(state, True)
    if op == "policy":
        return _plain_policy(state)
    return _plain_distill(state)


def _distinct(case):
    """How many different tokens a batch is expected to have."""
    p = np.log1p(1.0 / np.arange(1, case["v"] + 1)) / math.log(case["v"] + 1)
    return float((1 - np.exp(case["n"] * (1 - case["pad"]) * np.log1p(-p))).sum())


def work(case):
    n, v, op, e = case["n"], case["v"], case["op"], SIZE[case["dtype"]]
    if op == "lookup":
        return dict(bytes=n * 8 + (_distinct(case) + n) * case["d"] * e, flops=n * case["d"])
    if op == "grad":
        d, keep, to = case["d"], n * (1 - case["pad"]), SIZE[case["to"]]
        table = 2 * _distinct(case) * d * to if case["add"] else v * d * to
        return dict(bytes=n * 8 + keep * d * e + table, flops=keep * d)
    if op == "logprobs":
        return dict(bytes=n * v * e + n * (16 + 8 * case["k"]), flops=6 * n * v)
    if op == "policy":
        return dict(bytes=2 * n * v * e + n * 24, flops=14 * n * v)
    k = case["k"] * (0.5 if case["ragged"] else 1.0)
    return dict(bytes=(2 if case["grad"] else 1) * n * v * e + n * (16 + 8 * k), flops=(9 if case["grad"] else 4) * n * v)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op, n, v = case["op"], case["n"], case["v"]
    if op == "lookup":
        out = torch.zeros(n, case["d"], dtype=torch.float64, device="cuda")
        here = (s["tokens"] >= 0).nonzero()[:, 0]
        out[here] = torch.index_select(s["w"], 0, s["tokens"][here]).double().mul_(s["scale"])
        return out
    if op == "grad":   # the difference of running sums over the sorted tokens, some columns at a time
        tok, order = torch.sort(s["tokens"], stable=True)
        ends = torch.searchsorted(tok, torch.arange(-1, v, device="cuda"), right=True)
        out = torch.empty(v, case["d"], dtype=torch.float64, device="cuda")
        for lo in range(0, case["d"], 256):
            run_ = torch.cat([torch.zeros(1, min(256, case["d"] - lo), dtype=torch.float64, device="cuda"),
                              s["dy"][order, lo:lo + 256].double().cumsum(0)])
            out[:, lo:lo + 256] = (run_[ends[1:]] - run_[ends[:-1]]) * s["scale"]
        return out + s["dw"].double() if case["add"] else out
    parts, step = [], max(1, (1 << 25) // v)
    for lo in range(0, n, step):
        z = s["logits"][lo:lo + step].double() / case["temp"]
        rows = torch.arange(z.shape[0], device="cuda")
        logq = torch.log_softmax(z, 1)
        if op in ("logprobs", "policy"):
            tok = s["tokens"][lo:lo + step]
            plogp = torch.xlogy(logq.exp(), logq.exp())
            entropy = -plogp.sum(1)
            part = [logq[rows, tok], entropy]
            if op == "policy":
                q = logq.exp()
                hot = torch.zeros_like(q)
                hot[rows, tok] = 1.0
                g, h = s["g_logprob"][lo:lo + step, None].double(), s["g_entropy"][lo:lo + step, None].double()
                part.append((g * (hot - q) - h * (plogp + q * entropy[:, None])) / case["temp"])
            elif case["k"]:
                index = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : case["k"]]
                part += [index.to(torch.int32), logq.gather(1, index)]
        else:
            ptr = s["rowptr"][lo:lo + z.shape[0] + 1].tolist()
            row = torch.bucketize(torch.arange(ptr[0], ptr[-1], device="cuda"), s["rowptr"][lo + 1:lo + z.shape[0]], right=True)
            score = torch.full_like(z, -math.inf)
            score[row, s["col"][ptr[0]:ptr[-1]].long()] = s["val"][ptr[0]:ptr[-1]].double() / case["temp"]
            p = torch.softmax(score, 1).nan_to_num(0.0)   # a row without entries has no mass
            part = [(torch.xlogy(p, p) - torch.where(p > 0, p * logq, 0.0)).sum(1)]
            if case["grad"]:
                mass = p.sum(1, keepdim=True).round()
                part.append((mass * logq.exp() - p) * s["weight"][lo:lo + step, None].double() / case["temp"])
        parts.append(part)
    out = [torch.cat(p) for p in zip(*parts)]
    return out[0] if len(out) == 1 else tuple(out)
