"""Tokens from logits and given random numbers (cudatransformer_amd.sampling) against 64 bits."""
import math

import numpy as np
import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

gpu = pytest.mark.gpu


def reference(x, u, t, k, p, m):
    """(token, log-probability, distance of u from the nearest border) of one row, in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)) + 0.0
    top = x.max()
    if top == -np.inf:
        return -1, -math.inf, 1.0
    greedy = not t > 0
    t = 1.0 if greedy else t
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(x == top, 0.0, (x - top) / t)
        e = np.where(np.isnan(e), -np.inf, e)
    w = np.exp(e)
    order = np.argsort(-x, kind="stable")
    n = len(x) if k < 1 else min(k, len(x))
    if greedy:
        n = 1
    r = w[order[:n]]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(r)[:-1]])
        n = max(1, int((before < p * r.sum()).sum()))
    if m > 0:
        n = max(1, min(n, int((r >= m).sum())))
    mass = np.zeros_like(w)
    mass[order[:n]] = w[order[:n]]
    cum = np.cumsum(mass)
    target = float(u) * cum[-1]
    token = int(np.searchsorted(cum, target, side="right"))
    return token, e[token] - math.log(w.sum()), float(np.abs(cum / cum[-1] - float(u)).min())


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0, **kw):
    tokens, logprobs = ct.sample_tokens(logits, u, t, k, p, m, **kw)
    rows = logits.shape[0]
    each = lambda v: v.tolist() if isinstance(v, torch.Tensor) else [v] * rows  # noqa: E731
    x = logits.float().cpu().numpy()
    for i, (ui, ti, ki, pi, mi) in enumerate(zip(u.tolist(), each(t), each(k), each(p), each(m))):
        token, lp, near = reference(x[i], ui, ti, ki, pi, mi)
        where = f"row {i}: u={ui} t={ti} k={ki} p={pi} m={mi}"
        assert tokens[i].item() == token or near < 1e-11, f"{where}: token {tokens[i].item()}, expected {token}"
        if tokens[i].item() == token:
            # One rounding to 32 bits, of a sum that may be as large as the largest difference.
            assert math.isclose(logprobs[i].item(), lp, rel_tol=2**-23, abs_tol=1e-10), f"{where}: {logprobs[i].item()} {lp}"
    return tokens, logprobs


def logits_of(rows, vocab, dtype, seed, spread=2.0, sure=None):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((rows, vocab), generator=g)
    likely = min(64, max(1, vocab // 4))
    at = torch.randint(0, vocab, (rows, likely), generator=g)
    base = math.log(vocab) + (1.0 + 5.0 * torch.rand((rows, 1), generator=g) if sure is None else sure)
    x.scatter_(1, at, base - 0.3 * torch.arange(likely) + 0.3 * torch.randn((rows, likely), generator=g))
    return x.to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HOW = [dict(), dict(t=0.0), dict(t=0.7), dict(k=1), dict(k=7), dict(p=0.9), dict(p=0.5, t=1.3), dict(m=0.05), dict(k=50, p=0.9, m=0.02, t=0.8),
       dict(p=0.0), dict(m=2.0), dict(k=3, m=1.0), dict(p=0.999)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 65, 511, 513, 2048, 2049, 5003, 8192, 8193, 50257])
def test_against_64_bits(dtype, vocab):
    x, u = logits_of(9, vocab, dtype, vocab)
    for how in HOW:
        check(x, u, **how)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_nuclei(dtype):
    """Kept runs of thousands of tokens, more than are ranked at once: the histogram and its refinements."""
    for vocab, spread in ((20001, 1.0), (131072, 0.5), (131072, 3.0), (60000, 1e-3)):
        x, u = logits_of(5, vocab, dtype, vocab, spread, sure=-3.0)
        for how in (dict(p=0.9), dict(p=0.3), dict(k=5000), dict(k=9000, p=0.7), dict(k=9000, p=0.999, m=0.01), dict(m=1e-4), dict(k=vocab - 1),
                    dict(p=0.9, t=30.0), dict(p=0.95, t=0.05), dict(k=3000, m=0.5)):
            check(x, u, **how)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [100, 3000, 40000])
def test_ties(dtype, vocab):
    """Equal logits: the lower ids come first, also across the border of what is kept."""
    x = torch.zeros((6, vocab), dtype=dtype, device="cuda")
    x[1] = torch.arange(vocab, device="cuda") % 3
    x[2, ::2] = -0.0
    x[3, vocab // 2:] = 5.0
    x[4] = torch.randint(0, 4, (vocab,), generator=torch.Generator().manual_seed(1)).to(dtype)
    x[5, 7:] = -math.inf
    u = torch.tensor([0.0, 0.3, 0.9999999, 0.61, 0.12, 0.8], device="cuda")
    for how in (dict(), dict(t=0.0), dict(k=2), dict(k=vocab // 3), dict(p=0.371), dict(k=vocab // 2 + 1, p=0.77), dict(m=0.5), dict(m=1.0),
                dict(k=vocab // 2, p=0.5, m=0.1, t=2.0)):
        check(x, u, **how)


@gpu
@pytest.mark.parametrize("vocab", [9, 600, 30000])
def test_values_at_the_ends(vocab):
    """Masked tokens, NaN, infinities, the type's lowest value, and temperatures far from one."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn((8, vocab), generator=g)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, torch.randperm(vocab, generator=g)[:vocab - 2]] = -math.inf
    x[3, ::2] = math.nan
    x[4, 1], x[4, vocab - 1] = math.inf, math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6, 3:] = torch.finfo(torch.float32).min
    x[7] *= 1e30
    u = torch.tensor([0.5, 0.5, 0.5, 0.1, 0.7, 0.999, 0.3, 0.2]).cuda()
    for how in HOW + [dict(t=1e-30), dict(t=1e30), dict(t=math.inf), dict(t=math.nan), dict(p=math.nan, m=math.nan), dict(t=1e30, p=0.5),
                      dict(t=1e-30, k=5)]:
        check(x.cuda(), u, **how)
    tokens, logprobs = ct.sample_tokens(x.cuda(), u)
    assert tokens[:2].tolist() == [-1, -1] and logprobs[:2].tolist() == [-math.inf] * 2


@gpu
def test_random_numbers_at_the_ends():
    x, _ = logits_of(6, 3001, torch.float32, 4)
    last = float(np.nextafter(np.float32(1), np.float32(0)))
    for how in (dict(), dict(k=9), dict(p=0.9), dict(p=0.99, t=5.0)):
        check(x, torch.tensor([0.0, last, 1e-30, 0.5, 0.25, 0.75], device="cuda"), **how)
        # Numbers that are none of [0, 1) draw a kept token all the same.
        kept = ct.sample_tokens(x, torch.tensor([1.0, math.nan, -3.0, 7.0, math.inf, 1.0], device="cuda"), top_k=1)[0]
        assert torch.equal(kept, x.argmax(1))


@gpu
def test_parameters_of_each_row():
    x, u = logits_of(64, 30011, torch.bfloat16, 9)
    g = torch.Generator().manual_seed(2)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (64,), generator=g)].cuda()  # noqa: E731
    check(x, u, pick(0.0, 0.7, 1.0, 1.5), pick(0, 1, 5, 300, 4000).int(), pick(1.0, 0.2, 0.9, 0.98), pick(0.0, 0.01, 0.3))
    check(x, u, pick(0.0, 0.7, 1.0, 1.5), 20, pick(1.0, 0.2, 0.9, 0.98), 0.01)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_streams_graphs(dtype):
    """Rows of a longer tensor at odd places, another stream, given outputs and workspaces, captured and replayed."""
    whole, u = logits_of(12, 9001, dtype, 5)
    x = whole[:, 3:8804][::3]
    u = u[::3].contiguous()
    want = check(x, u, k=40, p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ct.sample_tokens(x, u, top_k=40, top_p=0.9, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    tokens, logprobs = torch.empty(4, dtype=torch.int64, device="cuda"), torch.empty(4, device="cuda")
    ws = torch.empty(ct.sample_workspace_bytes(4, 8801), dtype=torch.uint8, device="cuda")
    buf, draws = whole.clone(), u.clone()
    view = buf[:, 3:8804][::3]
    with torch.cuda.stream(side):
        ct.sample_tokens(view, draws, 0.8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ct.sample_tokens(view, draws, 0.8, 300, 0.95, 0.0, tokens=tokens, logprobs=logprobs, workspace=ws)
    for seed in range(4):
        new, un = logits_of(12, 9001, dtype, 50 + seed)
        buf.copy_(new)
        draws.copy_(un[::3])
        graph.replay()
        eager = check(view, draws, 0.8, 300, 0.95)
        torch.cuda.synchronize()
        assert torch.equal(tokens, eager[0]) and torch.equal(logprobs, eager[1])


@gpu
def test_frequencies():
    """Many draws follow the probabilities: every count within five standard deviations."""
    n = 60000
    z = torch.tensor([2.0, 0.0, 1.0, -1.0, 1.5, -30.0], device="cuda")
    u = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
    tokens, _ = ct.sample_tokens(z.expand(n, 6).contiguous(), u, 0.9, top_k=4)
    p = torch.where(torch.tensor([1, 1, 1, 0, 1, 0], dtype=torch.bool), torch.exp(z.cpu().double() / 0.9), 0.0)
    p /= p.sum()
    count = torch.bincount(tokens.cpu(), minlength=6).double()
    assert ((count - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p)) + 1e-9).all()


@gpu
def test_empty_and_large():
    none = ct.sample_tokens(torch.empty((0, 70), device="cuda"), torch.empty(0, device="cuda"))
    assert none[0].shape == none[1].shape == (0,)
    x, u = logits_of(2, 524288, torch.float32, 3)
    for how in (dict(), dict(k=50), dict(p=0.9)):
        check(x, u, **how)


@gpu
def test_refusals():
    x, u = torch.zeros((3, 20), device="cuda"), torch.zeros(3, device="cuda")
    f = ct.sample_tokens
    for call in (lambda: f(x.cpu(), u), lambda: f(x[0], u), lambda: f(x.double(), u), lambda: f(x.t(), u[:1]), lambda: f(x, u.cpu()),
                 lambda: f(x, u.double()), lambda: f(x, u[:2]), lambda: f(x), lambda: f(x, None, u), lambda: f(x, 0.5), lambda: f(x, u, u.double()),
                 lambda: f(x, u, top_k=u), lambda: f(x, u, top_p=u[:2]), lambda: f(x, u, min_p=u.int()), lambda: f(x, u, tokens=u),
                 lambda: f(x, u, logprobs=u.double()), lambda: f(torch.zeros((1, 524289), device="cuda"), u[:1]),
                 lambda: f(torch.zeros((65536, 1), device="cuda"), torch.zeros(65536, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        f(x, u, top_k=2.5)
    with pytest.raises(RuntimeError):
        f(x, u, logprobs=u)
    assert f(x, None, 0.0)[0].tolist() == [0, 0, 0]


def test_c_refusals():
    """What the entry point refuses before it touches memory."""
    lib = _capi.load()

    def call(dtype=0, logits=1 << 20, u=1 << 12, t=None, t_all=1.0, tokens=1 << 13, logprobs=1 << 14, ws=1 << 30, ws_bytes=1 << 20, rows=3,
             vocab=20000, stride=20000):
        return lib.ctattn_sample(dtype, logits, u, t, None, None, None, t_all, 0, 1.0, 0.0, tokens, logprobs, ws, ws_bytes, rows, vocab, stride,
                                 None)

    assert call(rows=0) == 0
    for kw in (dict(dtype=3), dict(dtype=8), dict(rows=-1), dict(rows=65536), dict(vocab=0), dict(vocab=1 << 20), dict(stride=19999),
               dict(logits=None), dict(u=None), dict(u=None, t_all=0.0, t=1 << 15), dict(tokens=None), dict(logprobs=None), dict(ws=None),
               dict(ws_bytes=5), dict(ws=(1 << 30) + 8), dict(tokens=1 << 12), dict(ws=1 << 20), dict(logprobs=1 << 13)):
        assert call(**kw) != 0, kw
    assert lib.ctattn_sample_workspace_bytes(-1, 5) == -1 and lib.ctattn_sample_workspace_bytes(5, 0) == -1


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1500, 20000, 131072])
def test_ranks_about_the_number_of_parts(dtype, vocab):
    """As many ranks as there are runs of 128 logits, one fewer and more; few tokens that are not masked; logits all below zero,
    of large values, in few places."""
    parts = 4 * -(-vocab // 512)
    x, u = logits_of(6, vocab, dtype, vocab + 1)
    x[1] -= 60.0  # all below zero
    x[2, torch.randperm(vocab, generator=torch.Generator().manual_seed(2))[:vocab - 5].cuda()] = -math.inf
    x[3, 300:] = -math.inf  # in three runs of 128
    x[4] *= 300.0
    x[5] = x[5].sort().values  # the largest behind each other
    for k in (128, parts - 1, parts, parts + 1, 511, 512, 513):
        for how in (dict(k=k), dict(k=k, p=0.7, t=3.0), dict(k=k, m=0.01)):
            check(x, u, **how)
    for how in (dict(p=0.3), dict(p=0.9, t=4.0), dict(m=1e-4, p=0.99)):
        check(x, u, **how)
