"""The range of fp16 in attention on packed sequences, against attention in 64 bits: gradients whose dS lies far
above or below what fp16 holds, while dQ, dK and dV are inside it.

The bounds are error bounds, computed beside the reference for every element, without an absolute term for dS: u = 2^-11
is half a step of fp16.  P and dS enter their second products rounded to fp16 and scaled by powers of two, so that half a
subnormal step is 2^-35 of P (2^-10 of 2^-25: P is at most 1) and 2^-32 of the largest |dS| of the row (dQ) or key (dK),
which lies at 2^7 or above.  Sums of n terms in fp32 are off by n 2^-24 of the terms' absolute sum, scores by d 2^-24
of theirs, and outputs are rounded once: by u of the value, or half a subnormal step, 2^-25.
"""
import math

import pytest
import torch

import cudatransformer_amd as ct

U, E = 2.0 ** -11, 2.0 ** -24
F16 = torch.float16


def _reference(q, k, v, do, lens, causal, eta_o):
    """{name: (value, bound)} in 64 bits; eta_o: half a subnormal step of the forward's P, of the row's sum."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    hkv, d = k.shape[1], k.shape[2]
    grp, c = q.shape[1] // hkv, 1 / math.sqrt(d)
    out = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    at = 0
    for n in lens:
        w = slice(at, at + n)
        at += n
        if n == 0:
            continue
        token = torch.arange(n, device=q.device)
        hide = token.repeat_interleave(grp)[:, None] < token[None] if causal else None
        for h in range(hkv):
            heads = slice(h * grp, (h + 1) * grp)
            a, g = (t[w, heads].reshape(n * grp, d) for t in (q, do))  # rows (token, head of the group)
            b, x = k[w, h], v[w, h]
            s, sa = a @ b.t() * c, a.abs() @ b.abs().t() * c
            if hide is not None:
                s, sa = s.masked_fill(hide, -math.inf), sa.masked_fill(hide, 0.0)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            es = (d + 4) * E * sa + 4 * E * (s.abs().masked_fill(s.abs() == math.inf, 0) + 64 + lse.abs())  # 64: scales' exponents
            ep = es + es.amax(1, keepdim=True) + (n + 16) * E  # P's, relative
            o = p @ x
            bo = (p * (ep + U + n * E) + eta_o) @ x.abs()
            bo = bo + U * (o.abs() + bo) + 2.0 ** -25
            dp = g @ x.t()
            delta, bdelta = (g * o).sum(1, keepdim=True), (g.abs() * (bo + d * E * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            rough = p * ((ep + U + 4 * E) * ((dp - delta).abs() + bdelta) + bdelta + (d + 4) * E * (g.abs() @ x.abs().t() + delta.abs()))
            small = lambda dim: 2.0 ** -32 * (ds.abs() + rough).amax(dim, keepdim=True)  # noqa: E731, B023
            terms = n * grp
            dq, dk, dv = ds @ b * c, ds.t() @ a * c, p.t() @ g
            bq = (rough + small(1) + n * E * (ds.abs() + rough)) @ b.abs() * c
            bk = (rough + small(0) + terms * E * (ds.abs() + rough)).t() @ a.abs() * c
            bv = (p * (ep + U + terms * E) + 2.0 ** -35).t() @ g.abs()
            last = lambda val, bound: bound + U * (val.abs() + bound) + 2.0 ** -25  # noqa: E731
            for name, part, val, bound in (("o", (w, heads), o, bo), ("dq", (w, heads), dq, last(dq, bq)),
                                           ("dk", (w, h), dk, last(dk, bk)), ("dv", (w, h), dv, last(dv, bv))):
                out[name][0][part] = val.reshape(out[name][0][part].shape)
                out[name][1][part] = bound.reshape(out[name][1][part].shape)
    return out


def _check(got, want):
    for name, t in got.items():
        val, bound = want[name]
        assert float(val.abs().max()) < 60000, f"{name}: the inputs leave fp16's range by themselves"
        assert torch.isfinite(t).all(), name
        err = (t.double() - val).abs()
        over = float((err - bound).max())
        assert over <= 0, f"{name}: {over:.3e} over the bound, error {float(err.max()):.3e}, values to {float(val.abs().max()):.3e}"


def _random(lens, hq, hkv, d, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((sum(lens), h, d), generator=g) for h in (hq, hkv, hkv, hq)]


def _position(lens):
    return torch.cat([torch.linspace(0, 1, n) if n > 1 else torch.zeros(n) for n in lens])[:, None, None]


def large(lens, hq, hkv, d):
    """dO as a loss scale leaves it: |dP| passes 65504."""
    q, k, v, do = _random(lens, hq, hkv, d, seed=d)
    return q / 4, k / 4, 4 * v, 5000 * do


def growing(lens, hq, hkv, d):
    """Later keys have far larger values and earlier rows far larger dO: what is largest grows all along either walk."""
    q, k, v, do = _random(lens, hq, hkv, d, seed=d + 1)
    at = _position(lens)
    return q, k, v * torch.exp2(18 * at - 10), do * torch.exp2(3 - 14 * at)


def small(lens, hq, hkv, d):
    """dO of an unscaled mean loss over long rows: every dS lies at a subnormal step or below.  V and half of K's columns
    change sign from key to key, half of Q's columns do not, so that dK and dQ are sums of like terms."""
    q, k, v, do = _random(lens, hq, hkv, d, seed=d + 2)
    sign = (1 - 2 * (torch.arange(sum(lens)) % 2))[:, None, None]
    half = torch.arange(d) < d // 2
    q = torch.where(half, 2 + 0.1 * q, 0 * q)
    k = torch.where(half, 0.02 * k, sign * (0.5 + 0.1 * k))
    return q, k, sign * (1 + 0.1 * v), 4e-6 * (1 + 0.1 * do)


SHORT = [1, 0, 33, 64, 65, 127, 2, 129, 200]
# By the kernels' shares of work: sequences that leave the chip short of work, and enough of them.
CASES = [(kind, lens, hq, hkv, d, causal)
         for d in (32, 64, 80, 128)
         for kind, lens, hq, hkv, causal in ((large, SHORT, 4, 1, True), (large, SHORT, 4, 2, False), (large, [256] * 40, 8, 4, True),
                                             (growing, SHORT, 4, 2, True), (growing, [700, 90], 4, 2, False),
                                             (growing, [256] * 40, 8, 4, False),
                                             (small, [4096], 1, 1, False), (small, [2048] * 4, 4, 4, False), (small, [3000], 4, 1, True))]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,lens,hq,hkv,d,causal", CASES)
def test_gradients(kind, lens, hq, hkv, d, causal):
    x = [t.to(F16).cuda() for t in kind(lens, hq, hkv, d)]
    plan = ct.packed_plan(lens, hq, hkv)
    o, lse = ct.flash_attn_packed_fwd(*x[:3], plan, causal=causal)
    dq, dk, dv = ct.flash_attn_packed_bwd(*x[:3], o, x[3], lse, plan, causal=causal)
    _check(dict(dq=dq, dk=dk, dv=dv), _reference(*x, lens, causal, eta_o=2.0 ** -25))


@pytest.mark.gpu
def test_an_infinity_in_one_row_of_do_stays_in_its_row_of_dq():
    lens, hq, hkv, d = [200, 90], 4, 2, 64
    x = [t.to(F16).cuda() for t in small(lens, hq, hkv, d)]
    want = _reference(*x, lens, True, eta_o=2.0 ** -25)
    plan = ct.packed_plan(lens, hq, hkv)
    o, lse = ct.flash_attn_packed_fwd(*x[:3], plan, causal=True)
    keep = torch.ones((sum(lens), hq), dtype=torch.bool, device="cuda")
    for at, value in (((100, 1), math.inf), ((40, 3), math.nan), ((230, 0), -math.inf)):
        x[3][at] = value
        keep[at] = False
    dq = ct.flash_attn_packed_bwd(*x[:3], o, x[3], lse, plan, causal=True)[0]
    assert not bool(torch.isfinite(dq[~keep]).any())
    _check(dict(dq=dq[keep]), dict(dq=tuple(t[keep] for t in want["dq"])))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,hq,hkv", [([8192], 1, 1), ([4096, 1000], 16, 4), ([700, 33], 4, 2)])
@pytest.mark.parametrize("gap", [12.0, 16.0, 17.05, 17.6])
def test_one_key_above_many(gap, lens, hq, hkv, causal):
    """One key's score lies e^gap above every other's: each of those has a P near or below a subnormal step of fp16, and all
    of them together make the output."""
    d, n = 64, sum(lens)
    q, k, v, _ = _random(lens, hq, hkv, d, seed=5)
    q, k, v = 0 * q, 0 * k, 1 + 0.1 * v
    q[:, :, 0] = 8
    for first in [sum(lens[:i]) for i in range(len(lens))]:
        k[first, :, 0], v[first] = gap, 0
    x = [t.to(F16).cuda() for t in (q, k, v)]
    o, _ = ct.flash_attn_packed_fwd(*x, ct.packed_plan(lens, hq, hkv), causal=causal)
    # P's rounding in the forward: 2^-32, half a subnormal step where the row's largest P is held at 2^7 or above.
    _check(dict(o=o), _reference(*x, torch.zeros_like(x[0]), lens, causal, eta_o=2.0 ** -32))
