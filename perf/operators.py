"""Operators of training a language model on packed documents, each in its plain form and as the
framework's call, over the ranges that users run.

``own`` chooses: False computes an operator with elementary torch operations in 32 bits (rounded
once at the end), True makes the framework's call.  ``listed()`` names the fixed cases,
``draw(rng)`` gives one more of the same ranges, ``prepare(case, seed)`` makes what a program
holds before the call, ``run(state)`` makes one pass, ``work(case)`` is the least a pass must move
and compute, and ``exact(case, seed)`` is the same result in 64 bits.

Three kinds of case:
  attn   attention on documents packed one behind the other, [tokens, heads, d], every document
         by itself, with fewer key / value heads than query heads; forward alone or with backward
  embed  the scaled lookup of token rows ("fwd") or the gradient of the table ("bwd")
  ortho  Newton-Schulz iteration that brings the singular values of an update near one
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_COEFFS = (3.4445, -4.7750, 2.0315)
_EPS = 1e-7


def listed():
    return [
        # Four short prompts of one serving batch, one of a single token: launches and latency.
        dict(name="attn-prompt-short", kind="attn", dtype="bf16", lens="1,7,33,60", hq=16, hkv=4, d=64, causal=True,
             train=False),
        # Prompts of ordinary and ragged lengths through wide heads, four query heads to a key head.
        dict(name="attn-prompt", kind="attn", dtype="bf16", lens="4000,2049,1111,700,255,64,13", hq=32, hkv=8, d=128,
             causal=True, train=False),
        # A training step's documents, most of them short, in a mid-sized model.
        dict(name="attn-train-docs", kind="attn", dtype="bf16",
             lens="3011,2048,1777,1290,1024,901,777,640,512,487,401,333,290,256,201,177,129,128,100,77,64,50,31,9,2,1",
             hq=16, hkv=4, d=64, causal=True, train=True),
        # Long-context training: one long document and what fills the batch behind it. The largest.
        dict(name="attn-train-long", kind="attn", dtype="bf16", lens="8192,4099,2500,1204,389", hq=32, hkv=8, d=128,
             causal=True, train=True),
        # The small GPT's attention (6 heads of 64, fp32) on packed documents instead of rows of 256.
        dict(name="attn-train-f32", kind="attn", dtype="f32", lens="1023,700,512,511,400,256,255,200,130,65,32,11,1",
             hq=6, hkv=6, d=64, causal=True, train=True),
        # Looking up a batch's tokens in a real tokenizer's table, scaled by the root of its width.
        dict(name="embed-fwd", kind="embed", dtype="bf16", tokens=16384, vocab=50257, width=768, train=False, pad=0.0),
        # The gradient of that table: frequent tokens many times, most rows never.
        dict(name="embed-bwd", kind="embed", dtype="bf16", tokens=16384, vocab=50257, width=768, train=True, pad=0.0),
        # A vocabulary of characters: every row is hot.
        dict(name="embed-bwd-chars", kind="embed", dtype="f32", tokens=4096, vocab=65, width=384, train=True, pad=0.0),
        # A large batch, a wide table and padding that no row belongs to.
        dict(name="embed-bwd-large", kind="embed", dtype="bf16", tokens=65536, vocab=131072, width=2048, train=True,
             pad=0.05),
        # The small GPT's 24 square attention matrices in one call.
        dict(name="ortho-small", kind="ortho", dtype="f32", batch=24, rows=384, cols=384),
        # One MLP matrix of a mid-sized model, its update kept in 16 bits.
        dict(name="ortho-mlp", kind="ortho", dtype="bf16", batch=1, rows=4096, cols=1024),
        # The same matrix of a wide model.
        dict(name="ortho-wide", kind="ortho", dtype="f32", batch=1, rows=2048, cols=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_attn(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    while True:
        hq, hkv = rng.choice([(4, 4), (6, 6), (8, 2), (8, 1), (12, 12), (12, 4), (14, 2), (16, 4), (16, 16), (32, 8)])
        longest = _log(rng, 1, 8192)
        lens = [_log(rng, 1, longest) for _ in range(_log(rng, 1, 40))] + [longest]
        case = dict(kind="attn", dtype=dtype, lens=",".join(map(str, lens)), hq=hq, hkv=hkv,
                    d=rng.choice([32, 64, 64, 64, 128, 128, 128, 40, 80, 96]), causal=rng.random() < 0.85,
                    train=rng.random() < 0.6)
        # fp32 is a small model's type.
        if sum(lens) <= 20000 and work(case)["flops"] <= (4e11 if dtype == "f32" else 2e12):
            return case


def _draw_embed(rng):
    while True:
        case = dict(kind="embed", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), tokens=_log(rng, 1, 65536),
                    vocab=_log(rng, 40, 131072), width=rng.choice([_log(rng, 32, 2048), 8 * _log(rng, 8, 256)]),
                    train=rng.random() < 0.7, pad=rng.choice([0.0, 0.0, 0.05]))
        if work(case)["bytes"] <= 8.0e8:
            return case


def _draw_ortho(rng):
    while True:
        case = dict(kind="ortho", dtype=rng.choice(["f32", "bf16", "f16"]), batch=_log(rng, 1, 24),
                    rows=_log(rng, 32, 4096), cols=_log(rng, 32, 8192))
        if work(case)["flops"] <= 5e11:
            return case


def draw(rng):
    return rng.choice([_draw_attn, _draw_attn, _draw_embed, _draw_ortho])(rng)


# ---- attn -----------------------------------------------------------------------------------


def _lens(c):
    return [int(x) for x in c["lens"].split(",")]


def _attn_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(_lens(c))
    heads = [c["hq"], c["hkv"], c["hkv"]] + ([c["hq"]] if c["train"] else [])
    return [torch.randn((n, h, c["d"]), generator=g, device="cuda").to(_DTYPES[c["dtype"]]) for h in heads]


def _attn_plain(q, k, v, do, lens, causal):
    """O and the log of the softmax's sum [tokens, heads], with do also dQ, dK, dV, in 32 bits."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    group, scale, dtype = hq // hkv, 1.0 / math.sqrt(d), q.dtype
    x = [t.float() for t in (q, k, v, do) if t is not None]
    outs = [torch.empty_like(x[0]), torch.empty_like(x[0][:, :, 0])]
    if do is not None:
        outs += [torch.empty_like(t) for t in x[:3]]
    start = 0
    for n in lens:
        part = slice(start, start + n)
        start += n
        # [key heads, group, tokens, d] of the queries beside [key heads, 1, tokens, d] of the keys.
        qs = x[0][part].view(n, hkv, group, d).permute(1, 2, 0, 3)
        ks, vs = (t[part].permute(1, 0, 2).unsqueeze(1) for t in x[1:3])
        s = torch.matmul(qs, ks.transpose(-1, -2)).mul_(scale)
        if causal:
            s.masked_fill_(torch.ones((n, n), dtype=torch.bool, device=q.device).triu_(1), -math.inf)
        top = s.amax(-1, keepdim=True)
        p = s.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(total)
        o = torch.matmul(p, vs)
        back = lambda t: t.permute(2, 0, 1, 3).reshape(n, hq, -1)  # noqa: E731
        outs[0][part] = back(o)
        outs[1][part] = back(top + total.log())[:, :, 0]
        if do is not None:
            g = x[3][part].view(n, hkv, group, d).permute(1, 2, 0, 3)
            # Sums over the group's query heads, which share the key head.
            outs[4][part] = torch.matmul(p.transpose(-1, -2), g).sum(1).permute(1, 0, 2)
            ds = torch.matmul(g, vs.transpose(-1, -2)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            outs[2][part] = back(torch.matmul(ds, ks))
            outs[3][part] = torch.matmul(ds.transpose(-1, -2), qs).sum(1).permute(1, 0, 2)
    return tuple(t if i == 1 else t.to(dtype) for i, t in enumerate(outs))


def _prepare_attn(c, seed):
    s = dict(kind="attn", x=_attn_inputs(c, seed), lens=_lens(c), causal=c["causal"], train=c["train"])
    if own:
        import cudatransformer_amd as ct

        # The batch's plan, which a program makes once for all of a model's layers and both directions.
        s["plan"] = ct.packed_plan(s["lens"], c["hq"], c["hkv"], device="cuda")
    return s


def _run_attn(s):
    q, k, v = s["x"][:3]
    do = s["x"][3] if s["train"] else None
    if not own:
        return _attn_plain(q, k, v, do, s["lens"], s["causal"])
    import cudatransformer_amd as ct

    o, lse = ct.flash_attn_packed_fwd(q, k, v, s["plan"], causal=s["causal"])
    if do is None:
        return o, lse
    return (o, lse) + ct.flash_attn_packed_bwd(q, k, v, o, do, lse, s["plan"], causal=s["causal"])


def _exact_attn(c, seed):
    x = [t.double() for t in _attn_inputs(c, seed)]
    q, k, v = x[:3]
    o, lse = torch.empty_like(q), torch.empty_like(q[:, :, 0])
    dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    group, at = c["hq"] // c["hkv"], 0
    for n in _lens(c):
        w = slice(at, at + n)
        at += n
        hide = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1) if c["causal"] else None
        for h in range(c["hq"]):
            a, b, e = q[w, h], k[w, h // group], v[w, h // group]
            s = a @ b.t() / math.sqrt(c["d"])
            if hide is not None:
                s = s.masked_fill(hide, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            o[w, h], lse[w, h] = p @ e, z
            if c["train"]:
                g = x[3][w, h]
                t = p * (g @ e.t() - (g * o[w, h]).sum(1)[:, None]) / math.sqrt(c["d"])
                dq[w, h] = t @ b
                dk[w, h // group] += t.t() @ a
                dv[w, h // group] += p.t() @ g
    return (o, lse, dq, dk, dv) if c["train"] else (o, lse)


def _work_attn(c):
    n, size = sum(_lens(c)), 4 if c["dtype"] == "f32" else 2
    pairs = sum(m * (m + 1) / 2 if c["causal"] else m * m for m in _lens(c))
    qs, ks = n * c["hq"] * c["d"] * size, n * c["hkv"] * c["d"] * size
    stats, fwd = 4 * n * c["hq"], 4.0 * pairs * c["hq"] * c["d"]
    if not c["train"]:
        return dict(bytes=2 * qs + 2 * ks + stats, flops=fwd)
    # Read q, k, v, do; write o, dq, dk, dv and the sums; five products backward to two forward.
    return dict(bytes=4 * qs + 4 * ks + stats, flops=3.5 * fwd)


# ---- embed ----------------------------------------------------------------------------------


def _embed_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    # Words of a text: the frequency falls with the rank, and a tokenizer's ids are in no such order.
    rank = 1.0 / (torch.arange(c["vocab"], device="cuda", dtype=torch.float64) + 2.7)
    cdf = torch.cumsum(rank / rank.sum(), 0)
    r = torch.searchsorted(cdf, torch.rand(c["tokens"], generator=g, device="cuda", dtype=torch.float64))
    ids = torch.randperm(c["vocab"], generator=g, device="cuda")[r.clamp_(max=c["vocab"] - 1)].to(torch.int32)
    if c["pad"] > 0:
        ids[torch.rand(c["tokens"], generator=g, device="cuda") < c["pad"]] = -1  # belongs to no row
    rows = c["tokens"] if c["train"] else c["vocab"]
    x = torch.randn((rows, c["width"]), generator=g, device="cuda").to(_DTYPES[c["dtype"]])
    return ids, x, math.sqrt(c["width"])


def _prepare_embed(c, seed):
    ids, x, scale = _embed_inputs(c, seed)
    return dict(kind="embed", ids=ids, x=x, scale=scale, vocab=c["vocab"], train=c["train"])


def _run_embed(s):
    ids, x, scale = s["ids"], s["x"], s["scale"]
    if own:
        import cudatransformer_amd as ct

        if s["train"]:
            return ct.embedding_grad(ids, x, s["vocab"], scale=scale)
        return ct.embedding_lookup(ids, x, scale=scale)
    inside = (ids >= 0) & (ids < s["vocab"])
    at = torch.where(inside, ids, 0).long()
    if s["train"]:
        grad = torch.zeros((s["vocab"], x.shape[1]), device=x.device)
        grad.index_add_(0, at, x.float() * inside[:, None])
        return (grad * scale).to(x.dtype)
    return (x[at].float() * (scale * inside)[:, None]).to(x.dtype)


def _exact_embed(c, seed):
    ids, x, scale = _embed_inputs(c, seed)
    if not c["train"]:
        out = torch.zeros((c["tokens"], c["width"]), dtype=torch.float64, device=x.device)
        keep = torch.nonzero(ids >= 0)[:, 0]
        out[keep] = x[ids[keep].long()].double() * scale
        return out
    grad = torch.zeros((c["vocab"], c["width"]), dtype=torch.float64, device=x.device)
    keep = torch.nonzero(ids >= 0)[:, 0]
    grad.index_add_(0, ids[keep].long(), x[keep].double())
    return grad * scale


def _work_embed(c):
    size = 4 if c["dtype"] == "f32" else 2
    rows = c["vocab"] if c["train"] else c["tokens"]  # looked-up rows are read at most once each
    read = c["tokens"] if c["train"] else min(c["tokens"], c["vocab"])
    return dict(bytes=4 * c["tokens"] + (rows + read) * c["width"] * size, flops=1.0 * c["tokens"] * c["width"])


# ---- ortho ----------------------------------------------------------------------------------


def _ortho_inputs(c, seed):
    # A gradient's spectrum: a few strong directions over a floor of noise.
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, m, n = c["batch"], c["rows"], c["cols"]
    k = max(1, min(m, n) // 8)
    strength = torch.exp(-4.0 * torch.arange(k, device="cuda") / k)
    left = torch.randn((b, m, k), generator=g, device="cuda") * strength
    right = torch.randn((b, k, n), generator=g, device="cuda")
    x = torch.matmul(left, right) / math.sqrt(k) + 0.3 * torch.randn((b, m, n), generator=g, device="cuda")
    return (1e-3 * x).to(_DTYPES[c["dtype"]])


def _prepare_ortho(c, seed):
    return dict(kind="ortho", x=_ortho_inputs(c, seed))


def _run_ortho(s):
    x = s["x"]
    if own:
        import cudatransformer_amd as ct

        return ct.newton_schulz(x, steps=5, coeffs=_COEFFS, eps=_EPS)
    a, b, c = _COEFFS
    tall = x.shape[1] > x.shape[2]
    y = x.float().transpose(1, 2).contiguous() if tall else x.float()
    y = y / (torch.sqrt((y * y).sum((1, 2), keepdim=True)) + _EPS)
    for _ in range(5):
        gram = torch.matmul(y, y.transpose(1, 2))
        y = a * y + torch.matmul(b * gram + c * torch.matmul(gram, gram), y)
    return (y.transpose(1, 2) if tall else y).to(x.dtype).contiguous()


def _exact_ortho(c, seed):
    # y p(y^T y) with p(t) = a + b t + c t^2, from the side that has the fewer columns.
    y = _ortho_inputs(c, seed).double()
    wide = c["cols"] > c["rows"]
    if wide:
        y = y.mT.contiguous()
    y /= y.flatten(1).norm(dim=1)[:, None, None] + _EPS
    for _ in range(5):
        gram = y.mT.contiguous() @ y
        poly = _COEFFS[2] * (gram @ gram) + _COEFFS[1] * gram
        poly.diagonal(dim1=1, dim2=2).add_(_COEFFS[0])
        y = y @ poly
    return y.mT.contiguous() if wide else y


def _work_ortho(c):
    r, n, size = min(c["rows"], c["cols"]), max(c["rows"], c["cols"]), 4 if c["dtype"] == "f32" else 2
    # A step: two symmetric products, of which half is enough, and one full.
    step = 1.0 * r * (r + 1) * n + 1.0 * r * (r + 1) * r + 2.0 * r * r * n
    return dict(bytes=2 * c["batch"] * r * n * size, flops=5 * c["batch"] * step)


_KINDS = {"attn": (_prepare_attn, _run_attn, _work_attn, _exact_attn),
          "embed": (_prepare_embed, _run_embed, _work_embed, _exact_embed),
          "ortho": (_prepare_ortho, _run_ortho, _work_ortho, _exact_ortho)}


def prepare(case, seed):
    return _KINDS[case["kind"]][0](case, seed)


def run(state):
    return _KINDS[state["kind"]][1](state)


def work(case):
    return _KINDS[case["kind"]][2](case)


def exact(case, seed):
    return _KINDS[case["kind"]][3](case, seed)
