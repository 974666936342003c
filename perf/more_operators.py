"""Operators of generating many continuations of shared prompts, each in its plain form and as the
framework's call, over the ranges that users run.

``own`` chooses: False computes an operator with elementary torch operations in 32 bits (64 for the
weights of sampling, rounded once at the end), True makes the framework's call.  ``listed()`` names
the fixed cases, ``draw(rng)`` gives one more of the same ranges, ``prepare(case, seed)`` makes what a
program holds before the call, ``run(state)`` makes one pass, ``work(case)`` is the least a pass must
move and compute, and ``exact(case, seed)`` is the same result in 64 bits.

Four kinds of case:
  attn    attention of every request to its group's prompt and to its own tokens, both in a paged
          cache; a group's requests share the prompt's keys and values
  sample  tokens from logits and given random numbers, by temperature, top-k, top-p and min-p
  pages   pages for a step's new tokens and where each token goes ("reserve"), or the pages of
          finished requests given back ("release")
  write   a step's keys and values into their places in the cache
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # Four samples of the small GPT (6 heads of 64, fp32) from one prompt: launches and latency.
        dict(name="attn-samples-few", kind="attn", dtype="f32", groups=1, samples=4, prefix=200, suffix=56, new=1, hq=6,
             hkv=6, d=64, page=16, layout="token"),
        # Rollouts: eight prompts of different length, sixteen samples of each, one token a step.
        dict(name="attn-rollouts", kind="attn", dtype="bf16", groups=8, samples=16, prefix=2000, suffix=1024, new=1, hq=32,
             hkv=8, d=128, page=16, layout="token"),
        # Questions of different length behind one document, fp16, as many key heads as query heads.
        dict(name="attn-questions", kind="attn", dtype="f16", groups=1, samples=24, prefix=4100, suffix=700, new=150, hq=16,
             hkv=16, d=64, page=32, layout="head"),
        # One long prompt and a large batch deep in its continuations. The largest.
        dict(name="attn-long-prompt", kind="attn", dtype="bf16", groups=1, samples=256, prefix=32768, suffix=2048, new=1,
             hq=32, hkv=8, d=128, page=64, layout="head"),
        # Characters of the small GPT, one temperature for all.
        dict(name="sample-chars", kind="sample", dtype="f32", rows=64, vocab=65, how="temperature"),
        # One sequence of a model with a real tokenizer: latency of top-k and top-p.
        dict(name="sample-one", kind="sample", dtype="bf16", rows=1, vocab=50257, how="top"),
        # A serving batch whose requests each have their own parameters, some greedy.
        dict(name="sample-batch", kind="sample", dtype="bf16", rows=256, vocab=131072, how="mixed"),
        # One decode step of an ordinary batch: a token each, a page for some.
        dict(name="pages-decode", kind="pages", op="reserve", requests=256, new=1, held=1500, page=16),
        # Many prompts admitted at once.
        dict(name="pages-admit", kind="pages", op="reserve", requests=2048, new=60, held=0, page=16),
        # A batch of which a third has finished.
        dict(name="pages-release", kind="pages", op="release", requests=1024, new=0, held=2000, page=16),
        # One token of each request into the cache.
        dict(name="write-decode", kind="write", dtype="bf16", rows=256, hkv=8, d=128, page=16, layout="token"),
        # The prompts of many requests into the cache.
        dict(name="write-prompts", kind="write", dtype="bf16", rows=40000, hkv=8, d=128, page=64, layout="head"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_attn(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    while True:
        hq, hkv = rng.choice([(4, 4), (6, 6), (8, 2), (8, 1), (12, 4), (14, 2), (16, 4), (16, 16), (32, 8)])
        new = rng.choice([1, 1, 1, 1, _log(rng, 2, 200)])
        case = dict(kind="attn", dtype=dtype, groups=rng.choice([1, 1, 1, _log(rng, 2, 16)]), samples=_log(rng, 1, 256),
                    prefix=_log(rng, 1, 32768), suffix=new + _log(rng, 1, 2048), new=new, hq=hq, hkv=hkv,
                    d=rng.choice([32, 64, 64, 64, 128, 128, 128, 40, 80, 96]), page=rng.choice([8, 16, 16, 32, 64, 128]),
                    layout=rng.choice(["token", "head"]))
        n = sum(_counts(case)[1])
        pairs = n * hq * (case["prefix"] + case["suffix"])
        # fp32 is a small model's type; the plain form holds all scores at once.
        if pairs <= 4e8 and work(case)["bytes"] <= 1.2e9 and work(case)["flops"] <= (4e10 if dtype == "f32" else 1.4e11):
            return case


def _draw_sample(rng):
    while True:
        case = dict(kind="sample", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=_log(rng, 1, 512),
                    vocab=_log(rng, 40, 160000), how=rng.choice(["temperature", "top", "top", "min", "mixed", "mixed"]))
        if work(case)["bytes"] <= 6.8e7:
            return case


def _draw_pages(rng):
    op = rng.choice(["reserve", "reserve", "release"])
    while True:
        case = dict(kind="pages", op=op, requests=_log(rng, 1, 4096), new=rng.choice([1, 1, _log(rng, 1, 300)]),
                    held=rng.choice([0, _log(rng, 1, 4000)]) if op == "reserve" else _log(rng, 1, 4000),
                    page=rng.choice([8, 16, 16, 32, 64, 128]))
        if case["requests"] * case["new"] <= 130000 and case["requests"] * case["held"] <= 4e6:
            return case


def _draw_write(rng):
    while True:
        hkv, d = rng.choice([(1, 128), (2, 64), (4, 64), (6, 64), (8, 128), (16, 64), (2, 80), (8, 96), (3, 40)])
        case = dict(kind="write", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=_log(rng, 1, 65536), hkv=hkv, d=d,
                    page=rng.choice([8, 16, 16, 32, 64, 128]), layout=rng.choice(["token", "head"]))
        if work(case)["bytes"] <= 3.2e8:
            return case


def draw(rng):
    return rng.choice([_draw_attn, _draw_attn, _draw_sample, _draw_sample, _draw_pages, _draw_write])(rng)


def _spread(i):
    """Numbers of [0, 1) without a pattern that a tile would meet, the same for every seed."""
    return (0.6180339887498949 * (i + 1)) % 1.0


def _pool(g, pages, page, hkv, d, dtype, layout):
    """A cache of pages, [pages, page, key heads, d]; with layout "head" a page holds its heads one behind the other."""
    shape = (pages, page, hkv, d) if layout == "token" else (pages, hkv, page, d)
    x = torch.randn(shape, generator=g, device="cuda").to(_DTYPES[dtype])
    return x if layout == "token" else x.transpose(1, 2)


# ---- attn -----------------------------------------------------------------------------------


def _counts(c):
    """Tokens of each prompt, new tokens of each request, and its own tokens with the new ones."""
    b = c["groups"] * c["samples"]
    prompts = [c["prefix"] - int(c["prefix"] / 4 * _spread(i)) if i else c["prefix"] for i in range(c["groups"])]
    new = [1 + int(c["new"] * _spread(i + 3)) for i in range(b)] if c["new"] > 1 else [1] * b
    lens = [n + int((c["suffix"] - n + 1) * _spread(i)) for i, n in enumerate(new)]
    return prompts, new, lens


def _attn_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    prompts, new, lens = _counts(c)
    page, groups, b = c["page"], c["groups"], len(lens)
    pp, mp = [-(-n // page) for n in prompts], -(-c["prefix"] // page)
    sp, ms = [-(-n // page) for n in lens], -(-c["suffix"] // page)
    total = sum(pp) + sum(sp) + 7
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    held = torch.tensor(pp + sp, device="cuda")
    first = held.cumsum(0) - held
    column = torch.arange(max(mp, ms), device="cuda")
    pages = torch.where(column < held[:, None], order[(first[:, None] + column).clamp_(max=total - 1)], -1)
    s = dict(kind="attn", new=new, samples=c["samples"])
    s["prefix_table"] = pages[:groups, :mp].contiguous()
    s["table"] = pages[groups:, :ms].contiguous()
    s["prefix_lens"] = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["starts"] = None
    if c["new"] > 1:
        s["starts"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s["q"] = torch.randn((sum(new), c["hq"], c["d"]), generator=g, device="cuda").to(_DTYPES[c["dtype"]])
    s["k"], s["v"] = (_pool(g, total, page, c["hkv"], c["d"], c["dtype"], c["layout"]) for _ in range(2))
    assert b == s["table"].shape[0]
    return s


def _attn_plain(s):
    q, k, v, new = s["q"], s["k"], s["v"], s["new"]
    hq, hkv, d, page = q.shape[1], k.shape[2], q.shape[2], k.shape[1]
    group, b, g, most = hq // hkv, s["lens"].shape[0], s["prefix_lens"].shape[0], max(new)
    dev = q.device
    # Requests with fewer new tokens than the most repeat their last one: rows [requests, most].
    n = torch.ones(b, dtype=torch.int64, device=dev) if s["starts"] is None else s["starts"].diff().long()
    first = n.cumsum(0) - n
    token = torch.arange(most, device=dev)
    rows = first[:, None] + torch.minimum(token, n[:, None] - 1)
    x = q[rows].float().view(b, most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, most * group, d)

    def pages(cache, table):  # [tables, key heads, keys, d]
        return cache[table.clamp(min=0).long()].flatten(1, 2).transpose(1, 2).float()

    # A group's rows beside its prompt: one product for all of them.
    per = b // g
    xg = x.view(g, per, hkv, most * group, d).transpose(1, 2).reshape(g, hkv, per * most * group, d)
    kp, vp = pages(k, s["prefix_table"]), pages(v, s["prefix_table"])
    sp = torch.matmul(xg, kp.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    hide = torch.arange(kp.shape[2], device=dev) >= s["prefix_lens"][:, None]
    sp.masked_fill_(hide[:, None, None, :], -math.inf)
    # Every request beside its own tokens, up to each row's own place.
    ks, vs = pages(k, s["table"]), pages(v, s["table"])
    so = torch.matmul(x, ks.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    seen = s["lens"][:, None] - n[:, None] + torch.minimum(token, n[:, None] - 1) + 1
    hide = torch.arange(ks.shape[2], device=dev) >= seen.repeat_interleave(group, 1)[:, :, None]
    so.masked_fill_(hide[:, None], -math.inf)
    back = lambda t: t.view(g, hkv, per, most * group, -1).transpose(1, 2).reshape(b, hkv, most * group, -1)  # noqa: E731
    to = lambda t: t.view(g, per, hkv, most * group, -1).transpose(1, 2).reshape(g, hkv, per * most * group, -1)  # noqa: E731
    top = torch.maximum(back(sp.amax(-1, keepdim=True)), so.amax(-1, keepdim=True))
    p, r = sp.sub_(to(top)).exp_(), so.sub_(top).exp_()
    total = back(p.sum(-1, keepdim=True)) + r.sum(-1, keepdim=True)
    o = (back(torch.matmul(p, vp)) + torch.matmul(r, vs)) / total
    lse = top + total.log()
    # Rows [requests, most] to the tokens that there are.
    at = torch.arange(q.shape[0], device=dev)
    i = torch.searchsorted(first, at, right=True) - 1
    t = at - first[i]
    o = o.view(b, hkv, most, group, d).transpose(1, 2).reshape(b, most, hq, d)[i, t]
    lse = lse.view(b, hkv, most, group).transpose(1, 2).reshape(b, most, hq)[i, t]
    return o.to(q.dtype), lse


def _run_attn(s):
    if not own:
        return _attn_plain(s)
    import cudatransformer_amd as ct

    return ct.flash_attn_shared_prefix(s["q"], s["k"], s["v"], s["table"], s["lens"], s["prefix_table"], s["prefix_lens"],
                                       starts=s["starts"])


def _exact_attn(c, seed):
    s = _attn_inputs(c, seed)
    prompts, new, lens = _counts(c)
    group, d, page = c["hq"] // c["hkv"], c["d"], c["page"]
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")

    def keys(cache, table, n):  # [key heads, n, d]
        at = torch.arange(n, device="cuda")
        return cache[table.long()[at // page], at % page].double().transpose(0, 1).contiguous()

    row = 0
    for i, (n, own_tokens) in enumerate(zip(new, lens)):
        gi = i // c["samples"]
        if i % c["samples"] == 0:
            kp, vp = (keys(s[x], s["prefix_table"][gi], prompts[gi]) for x in "kv")
        ks, vs = (keys(s[x], s["table"][i], own_tokens) for x in "kv")
        x = s["q"][row:row + n].double().view(n, c["hkv"], group, d).permute(1, 0, 2, 3).reshape(c["hkv"], n * group, d)
        z = torch.cat([x @ kp.mT.contiguous(), x @ ks.mT.contiguous()], 2) / math.sqrt(d)
        last = torch.arange(n, device="cuda") + (prompts[gi] + own_tokens - n)
        z.masked_fill_(torch.arange(z.shape[2], device="cuda") > last.repeat_interleave(group)[:, None], -math.inf)
        total = torch.logsumexp(z, 2)
        p = torch.exp(z - total[:, :, None])
        y = p[:, :, :prompts[gi]].contiguous() @ vp + p[:, :, prompts[gi]:].contiguous() @ vs
        o[row:row + n] = y.view(c["hkv"], n, group, d).transpose(0, 1).reshape(n, c["hq"], d)
        lse[row:row + n] = total.view(c["hkv"], n, group).transpose(0, 1).reshape(n, c["hq"])
        row += n
    return o, lse


def _work_attn(c):
    prompts, new, lens = _counts(c)
    size, n = 4 if c["dtype"] == "f32" else 2, sum(new)
    pairs = sum(m * prompts[i // c["samples"]] + sum(range(s - m + 1, s + 1)) for i, (m, s) in enumerate(zip(new, lens)))
    cached = 2 * (sum(prompts) + sum(lens)) * c["hkv"] * c["d"] * size
    return dict(bytes=2 * n * c["hq"] * c["d"] * size + 4 * n * c["hq"] + cached, flops=4.0 * pairs * c["hq"] * c["d"])


# ---- sample ---------------------------------------------------------------------------------


def _sample_inputs(c, seed):
    # A trained model's logits: a broad bulk, and some tens of tokens above it by as much as the model is sure.
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, vocab = c["rows"], c["vocab"]
    x = 2.0 * torch.randn((n, vocab), generator=g, device="cuda")
    likely = min(64, max(1, vocab // 4))
    at = torch.randint(0, vocab, (n, likely), generator=g, device="cuda")
    sure = math.log(vocab) + 1.0 + 5.0 * torch.rand((n, 1), generator=g, device="cuda")
    value = sure - 0.3 * torch.arange(likely, device="cuda") + 0.3 * torch.randn((n, likely), generator=g, device="cuda")
    x.scatter_reduce_(1, at, value, "amax")
    logits = x.to(_DTYPES[c["dtype"]])
    u = torch.rand(n, generator=g, device="cuda")
    how = c["how"]
    if how == "mixed":  # every request its own
        pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (n,), generator=g, device="cuda")]  # noqa: E731
        kw = dict(temperature=pick(0.0, 0.6, 0.8, 1.0, 1.0, 1.3), top_k=pick(0, 0, 1, 20, 50, 200).to(torch.int32),
                  top_p=pick(1.0, 0.5, 0.9, 0.95), min_p=pick(0.0, 0.0, 0.02, 0.1))
    else:
        kw = dict(temperature=0.8, top_k=50 if how == "top" else 0, top_p=0.9 if how == "top" else 1.0,
                  min_p=0.05 if how == "min" else 0.0)
    return dict(kind="sample", logits=logits, u=u, kw=kw)


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    n, vocab = logits.shape
    each = lambda v: (v if isinstance(v, torch.Tensor) else torch.full((n,), v, dtype=torch.float64, device=logits.device))[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p = each(temperature).double(), each(top_k), each(top_p).double(), each(min_p).double()
    x = logits.float()
    greedy = temperature <= 0
    t = torch.where(greedy, 1.0, temperature)
    top = x.amax(1, keepdim=True)
    w = torch.exp((x.double() - top) / t)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    rank = torch.arange(vocab, device=x.device)
    most = torch.where(greedy, 1, torch.where(top_k > 0, top_k, vocab))
    first = torch.where(rank < most, ranked, 0.0)
    upto = first.cumsum(1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], 1)
    keep = (rank < most) & (before < torch.where(top_p >= 1, math.inf, top_p) * first.sum(1, keepdim=True)) & (ranked >= min_p)
    keep |= rank == 0
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0.0)).cumsum(1)
    token = (mass <= u[:, None].double() * mass[:, -1:]).sum(1)
    logprob = (x.gather(1, token[:, None]).double() - top) / t - w.sum(1, keepdim=True).log()
    return token, logprob[:, 0].float()


def _run_sample(s):
    if not own:
        return _sample_plain(s["logits"], s["u"], **s["kw"])
    import cudatransformer_amd as ct

    return ct.sample_tokens(s["logits"], s["u"], **s["kw"])


def _exact_sample(c, seed):
    s = _sample_inputs(c, seed)
    n = c["rows"]
    kw = {k: v.tolist() if isinstance(v, torch.Tensor) else [v] * n for k, v in s["kw"].items()}
    tokens, logprobs = [], []
    for i in range(n):
        x, t = s["logits"][i].double(), kw["temperature"][i]
        z = x if t <= 0 else x / t
        lp = z - torch.logsumexp(z, 0)
        down = torch.argsort(x, descending=True, stable=True)
        m = 1 if t <= 0 else kw["top_k"][i] or len(x)
        p = torch.exp(lp[down[:m]])
        if kw["top_p"][i] < 1:
            p = p[:1 + int((p.cumsum(0)[:-1] < kw["top_p"][i] * p.sum()).sum())]
        p = p[:max(1, int((p >= kw["min_p"][i] * p[0]).sum()))]
        ids, back = torch.sort(down[:len(p)])
        q = p[back].cumsum(0)
        tokens.append(ids[(q > s["u"][i].double() * q[-1]).to(torch.int8).argmax()])
        logprobs.append(lp[tokens[-1]])
    return torch.stack(tokens), torch.stack(logprobs)


def _work_sample(c):
    size = 4 if c["dtype"] == "f32" else 2
    # A difference, a scale, an exponential and a sum a logit.
    return dict(bytes=c["rows"] * (c["vocab"] * size + 32), flops=4.0 * c["rows"] * c["vocab"])


# ---- pages ----------------------------------------------------------------------------------


def _page_counts(c):
    """Own tokens of each request before the step, its new ones, and its first position's offset."""
    b = c["requests"]
    lens = [int((c["held"] + 1) * _spread(i)) for i in range(b)]
    new = [1] * b if c["new"] == 1 else [int((2 * c["new"] + 1) * _spread(i + 5)) for i in range(b)]
    return lens, new


def _prepare_pages(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, new = _page_counts(c)
    page, b = c["page"], c["requests"]
    held = [-(-n // page) for n in lens]
    most = max(1, -(-(c["held"] + 2 * c["new"] + 1) // page))
    need = sum(-(-(n + m) // page) for n, m in zip(lens, new))
    total = max(need, sum(held)) + 64
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    h = torch.tensor(held, device="cuda")
    first, column = h.cumsum(0) - h, torch.arange(most, device="cuda")
    table = torch.where(column < h[:, None], order[(first[:, None] + column).clamp_(max=total - 1)], -1)
    # The ring of free pages, somewhere in its life: what is free begins at `taken`.
    free = total - sum(held)
    taken = total * 1000 + int(total * _spread(seed % 1000))
    ring = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    ring[(taken + torch.arange(free, device="cuda")) % total] = order[sum(held):]
    return dict(kind="pages", op=c["op"], page=page, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                new=torch.tensor(new, dtype=torch.int32, device="cuda"), table=table, free=ring,
                counters=torch.tensor([taken, taken + free], device="cuda"),
                done=torch.rand(b, generator=g, device="cuda") < 0.33, tokens=sum(new) + 5,
                offsets=torch.randint(0, 30000, (b,), generator=g, device="cuda").to(torch.int32))


def _run_pages(s):
    lens, new, table, free, counters, page = s["lens"], s["new"], s["table"], s["free"], s["counters"], s["page"]
    if own:
        import cudatransformer_amd as ct

        if s["op"] == "release":
            return (free,) + ct.page_release(s["done"], lens, table, free, counters, page)
        return (table,) + ct.page_reserve(lens, new, table, free, counters, page, s["tokens"], offsets=s["offsets"])
    held = (lens + page - 1) // page
    ring, column = free.shape[0], torch.arange(table.shape[1], device=lens.device)
    if s["op"] == "release":
        back = torch.where(s["done"], held, 0).long()
        upto = back.cumsum(0)
        # Every ring place that a page comes back to, and the others as they were.
        place = (torch.arange(ring, device=lens.device) - counters[1]) % ring
        i = torch.searchsorted(upto, place, right=True).clamp_(max=lens.shape[0] - 1)
        page_of = table[i, (place - (upto - back)[i]).clamp(0, table.shape[1] - 1)]
        free.copy_(torch.where(place < upto[-1], page_of, free))
        return free, torch.where(s["done"], 0, lens), torch.stack([counters[0], counters[1] + upto[-1]])
    most = s["tokens"]
    total = lens + new
    pages = (total + page - 1) // page
    starts = torch.cat([new.new_zeros(1), new.cumsum(0).to(torch.int32)])
    fits = (pages <= table.shape[1]) & (starts[1:] <= most)
    need = torch.where(fits, pages - held, 0).long()
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= counters[1] - counters[0]))
    fresh = ok[:, None] & (column >= held[:, None]) & (column < pages[:, None])
    at = (counters[0] + (upto - need)[:, None] + column - held[:, None]) % ring
    table.copy_(torch.where(fresh, free[at], table))
    row = torch.arange(most, device=lens.device)
    i = torch.searchsorted(starts, row, right=True) - 1
    there = (row < starts[-1]) & ok[i.clamp(max=lens.shape[0] - 1)]
    i = i.clamp_(max=lens.shape[0] - 1)
    pos = lens[i].long() + row - starts[i]
    slot = table[i, (pos // page).clamp_(0, table.shape[1] - 1)].long() * page + pos % page
    taken = counters[0] + torch.where(ok, need, 0).sum()
    return (table, torch.where(there, slot, -1), torch.where(there, pos + s["offsets"][i], 0), starts,
            torch.where(ok, total, lens), torch.stack([taken, counters[1]]))


def _exact_pages(c, seed):
    return None  # whole numbers


def _work_pages(c):
    lens, new = _page_counts(c)
    page = c["page"]
    if c["op"] == "release":
        return dict(bytes=c["requests"] * 9 + 8 * sum(-(-n // page) for n in lens) * 0.33, flops=1.0 * c["requests"])
    fresh = sum(-(-(n + m) // page) - -(-n // page) for n, m in zip(lens, new))
    return dict(bytes=20 * c["requests"] + 16 * sum(new) + 8 * fresh, flops=1.0 * sum(new))


# ---- write ----------------------------------------------------------------------------------


def _prepare_write(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, page = c["rows"], c["page"]
    pages = -(-n * 5 // (4 * page)) + 1
    dtype = _DTYPES[c["dtype"]]
    k_cache, v_cache = (_pool(g, pages, page, c["hkv"], c["d"], c["dtype"], c["layout"]) for _ in range(2))
    # Keys and values as one projection leaves them, side by side; tokens in pages of no order, the last rows padding.
    kv = torch.randn((n, 2, c["hkv"], c["d"]), generator=g, device="cuda").to(dtype)
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = order[at // page] * page + at % page
    slots[1 + n - max(1, n // 50):] = -1
    return dict(kind="write", k=kv[:, 0], v=kv[:, 1], k_cache=k_cache, v_cache=v_cache, slots=slots)


def _run_write(s):
    k, v, k_cache, v_cache, slots = s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"]
    if own:
        import cudatransformer_amd as ct

        ct.cache_write(k, v, k_cache, v_cache, slots)
        return k_cache, v_cache
    # A row without a place repeats the first, which has one.
    there = slots >= 0
    at = torch.where(there, slots, slots[0])
    page = k_cache.shape[1]
    for cache, x in ((k_cache, k), (v_cache, v)):
        cache[at // page, at % page] = torch.where(there[:, None, None], x, x[0])
    return k_cache, v_cache


def _exact_write(c, seed):
    s = _prepare_write(c, seed)
    there = torch.nonzero(s["slots"] >= 0)[:, 0]
    out = []
    for cache, x in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        flat = cache.double().reshape(-1, c["hkv"], c["d"])
        flat[s["slots"][there]] = x[there].double()
        out.append(flat.view(cache.shape))
    return tuple(out)


def _work_write(c):
    size = 4 if c["dtype"] == "f32" else 2
    return dict(bytes=c["rows"] * (8 + 4 * c["hkv"] * c["d"] * size), flops=0.0)


_KINDS = {"attn": (_attn_inputs, _run_attn, _work_attn, _exact_attn),
          "sample": (_sample_inputs, _run_sample, _work_sample, _exact_sample),
          "pages": (_prepare_pages, _run_pages, _work_pages, _exact_pages),
          "write": (_prepare_write, _run_write, _work_write, _exact_write)}


def prepare(case, seed):
    return _KINDS[case["kind"]][0](case, seed)


def run(state):
    return _KINDS[state["kind"]][1](state)


def work(case):
    return _KINDS[case["kind"]][2](case)


def exact(case, seed):
    return _KINDS[case["kind"]][3](case, seed)
