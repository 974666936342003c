"""Attention on packed sequences: the plan, the refusals (CPU) and the kernels against attention in
64 bits, sequence by sequence (GPU).

The bounds are error bounds, computed beside the reference for every element: with u16 half a step of
the 16-bit type (0 in fp32), P and dS rounded once to that type as operands of the second products,
fp32 sums of n terms off by n 2^-24 of the terms' absolute sum, the scores by d 2^-24 of theirs (which
moves P by as much, relatively, and once more through the row's sum), outputs rounded once.  A
relative half step holds down to the smallest normal number alone: below it P and dS are off by up
to that number (2^-126 in fp32 and bf16; 2^-25, half a subnormal step, in fp16), each.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

# ---- the plan (host) ------------------------------------------------------------------------

TILE = [32, 64, 128, 32, 64, 128]  # rows of (token, head of the group) three times, then keys


def _plan_tables(lens, group):
    lib = _capi.load()
    arr = (ctypes.c_int64 * max(len(lens), 1))(*lens)
    need = lib.ctattn_packed_plan_bytes(arr, len(lens), group)
    assert need > 0
    buf = np.zeros(need, dtype=np.uint8)
    assert lib.ctattn_packed_plan(arr, len(lens), group, buf.ctypes.data, need) == 0
    head = buf[:512].view(np.int64)
    cu = buf[head[6]:head[6] + 4 * (len(lens) + 1)].view(np.int32)
    tables = []
    for i in range(12):
        at, count = head[9 + 2 * i], head[10 + 2 * i]
        assert at % 16 == 0 and at + 16 * count <= need
        tables.append(buf[at:at + 16 * count].view(np.int32).reshape(-1, 4))
    return head, cu, tables


@pytest.mark.parametrize("lens,group", [([5], 1), ([1, 0, 300, 64, 65, 0], 4), ([], 2), ([0, 0], 3), ([1000, 7, 129], 7)])
def test_plan_covers_every_tile_once(lens, group):
    head, cu, tables = _plan_tables(lens, group)
    assert list(head[2:6]) == [len(lens), sum(lens), max(lens, default=0), group]
    assert list(head[7:9]) == [sum(n * n for n in lens), sum(n * (n + 1) // 2 for n in lens)]
    assert list(cu) == list(np.concatenate([[0], np.cumsum(lens)]).astype(int))
    for i, table in enumerate(tables):
        causal, kind = divmod(i, 6)
        rows = [n if kind >= 3 else n * group for n in lens]
        want = {(int(cu[s]), lens[s], t, s) for s in range(len(lens)) for t in range(-(-rows[s] // TILE[kind]))}
        assert {tuple(x) for x in table.tolist()} == want and len(table) == len(want)
        # The longest running first.
        if not causal:
            cost = table[:, 1]
        elif kind >= 3:
            cost = table[:, 1] - table[:, 2] * TILE[kind]
        else:
            cost = np.minimum(table[:, 1], (table[:, 2] * TILE[kind] + TILE[kind] - 1) // group + 1)
        assert np.all(np.diff(cost) <= 0)


def test_plan_refusals():
    lib = _capi.load()
    one = lambda *x: (ctypes.c_int64 * len(x))(*x)  # noqa: E731
    for lens, group in [((-1,), 1), ((5,), 0), ((5,), 4097), ((1 << 31,), 1), ((1 << 30, 1 << 30, 1 << 30), 1), ((1 << 29,), 8)]:
        assert lib.ctattn_packed_plan_bytes(one(*lens), len(lens), group) == -1
    assert lib.ctattn_packed_plan_bytes(None, 2, 1) == -1
    assert lib.ctattn_packed_plan_bytes(one(1), -1, 1) == -1
    assert lib.ctattn_packed_plan(one(5), 1, 1, None, 1 << 20) == 1
    buf = (ctypes.c_char * 64)()
    assert lib.ctattn_packed_plan(one(5), 1, 1, ctypes.addressof(buf), 64) == 1
    assert "too small" in _capi.last_error()
    with pytest.raises(ValueError):
        ct.packed_plan([3, -1], 4, 2, device="cpu")
    with pytest.raises(ValueError):
        ct.packed_plan([3], 4, 3, device="cpu")
    with pytest.raises(ValueError):
        ct.packed_plan(torch.tensor([3.0]), 4, 2, device="cpu")


def test_c_entry_refusals():
    """Every bad argument is refused on the host, before any launch."""
    lib = _capi.load()
    plan = ct.packed_plan([5, 3], 4, 2, device="cpu")
    host = plan._host.data_ptr()
    st8 = (ctypes.c_int64 * 16)(*([256, 64, 128, 64, 128, 64, 256, 64] + [256, 64, 256, 64, 128, 64, 128, 64]))

    def fwd(dtype=1, p=64, strides=st8, host=host, dev=64, rows=8, hq=4, hkv=2, d=64):
        return lib.ctattn_packed_fwd(dtype, p, p, p, p, None, strides, host, dev, rows, hq, hkv, d, 1, None)

    bad = ctypes.create_string_buffer(4096)
    assert fwd(dtype=4) == 1 and fwd(host=None) == 1 and fwd(host=ctypes.addressof(bad)) == 1
    assert fwd(dev=None) == 1 and fwd(rows=7) == 1 and fwd(hq=3) == 1 and fwd(hq=8) == 1 and fwd(hkv=0) == 1
    assert fwd(d=0) == 801 and fwd(d=257) == 801 and fwd(strides=None) == 1 and fwd(p=None) == 1
    for o_row, o_head in [(256, 32), (64, 64), (0, 64), (256, 0), (-256, 64)]:
        st = (ctypes.c_int64 * 8)(256, 64, 128, 64, 128, 64, o_row, o_head)
        assert fwd(strides=st) == 1 and "overlap" in _capi.last_error()
    big = 1 << 20  # apart from each other
    call = lambda q, k, v, o: lib.ctattn_packed_fwd(1, q, k, v, o, None, st8, host, None, 8, 4, 2, 64, 1, None)  # noqa: E731
    assert call(big, 2 * big, 3 * big, 4 * big) == 1 and "device plan" in _capi.last_error()
    need = lib.ctattn_packed_bwd_workspace_bytes(1, host, 4, 2, 64)
    assert need > 0 and lib.ctattn_packed_bwd_workspace_bytes(1, host, 4, 4, 64) == -1

    def bwd(ws=256, size=need, p=64):
        return lib.ctattn_packed_bwd(1, p, p, p, p, p, p, p, p, p, ws, size, st8, host, 64, 8, 4, 2, 64, 1, None)

    assert bwd(p=None) == 1

    def grads(at, ws=256, size=need):
        return lib.ctattn_packed_bwd(1, *[a * big for a in at], 9 * big, *[a * big for a in (6, 7, 8)], ws, size, st8, host, 64, 8, 4,
                                     2, 64, 1, None)

    assert grads((1, 2, 3, 4, 5), ws=None) == 1 and grads((1, 2, 3, 4, 5), size=need - 1) == 1 and grads((1, 2, 3, 4, 5), ws=8) == 1
    for at in ((6, 2, 3, 4, 5), (1, 7, 3, 4, 5), (1, 2, 8, 4, 5), (1, 2, 3, 6, 5), (1, 2, 3, 4, 7)):
        assert grads(at) == 1 and "input's memory" in _capi.last_error()
    # Slices of one row-major buffer do not overlap, shifted ones do.
    wide = lambda o: lib.ctattn_packed_fwd(1, big, 4 * big, 4 * big, big + o, None, (ctypes.c_int64 * 8)(512, 64, 128, 64, 128, 64, 512, 64),  # noqa: E731
                                           host, 64, 8, 4, 2, 300, 1, None)
    assert wide(512) == 801  # the head dim is refused first
    with pytest.raises(ValueError, match="on the GPU"):
        ct.flash_attn_packed_fwd(torch.zeros(8, 4, 64), torch.zeros(8, 2, 64), torch.zeros(8, 2, 64), plan)


# ---- the kernels (GPU) ----------------------------------------------------------------------

gpu = pytest.mark.gpu


def _inputs(lens, hq, hkv, d, dtype, seed=0, extra=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens) + extra
    return [(scale * torch.randn((n, h, d), generator=g)).to(dtype).cuda() for h in (hq, hkv, hkv, hq)]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _reference(q, k, v, do, lens, causal):
    """{name: (value, bound)} in 64 bits."""
    dtype = q.dtype
    u16 = _half_step(dtype) if dtype in (torch.bfloat16, torch.float16) else 0.0
    uo = _half_step(dtype)
    e = 2.0 ** -24 if dtype != torch.float64 else 2.0 ** -52
    eta = {torch.float16: 2.0 ** -25, torch.float64: 2.0 ** -1022}.get(dtype, 2.0 ** -126)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    grp, c = hq // hkv, 1 / math.sqrt(d)
    z = lambda t: torch.zeros_like(t)  # noqa: E731
    out = {n: (z(t), z(t)) for n, t in (("o", q), ("lse", q[:, :, 0]), ("dq", q), ("dk", k), ("dv", v))}
    at = 0
    for n in lens:
        w = slice(at, at + n)
        at += n
        if n == 0:
            continue
        hide = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1) if causal else None
        for h in range(hq):
            a, b, x, g = q[w, h], k[w, h // grp], v[w, h // grp], do[w, h]
            s, sa = a @ b.t() * c, a.abs() @ b.abs().t() * c
            if hide is not None:
                s = s.masked_fill(hide, -math.inf)
                sa = sa.masked_fill(hide, 0.0)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            es = (d + 4) * e * sa + 4 * e * (s.abs().masked_fill(s.abs() == math.inf, 0) + lse.abs())  # a score's, and exp2's argument's
            ep = es + es.amax(1, keepdim=True) + (n + 16) * e  # P's, relative
            o, pv = p @ x, p @ x.abs()
            bo = (p * (ep + u16 + n * e) + eta) @ x.abs()
            out["o"][0][w, h], out["o"][1][w, h] = o, bo + uo * (o.abs() + bo)
            out["lse"][0][w, h] = lse[:, 0]
            out["lse"][1][w, h] = es.amax(1) + (n + 16) * e + 8 * e * lse.abs()[:, 0]
            dp = g @ x.t()
            delta = (g * o).sum(1, keepdim=True)
            bdelta = (g.abs() * (out["o"][1][w, h] + d * e * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            bds = p * ((ep + u16 + 4 * e) * ((dp - delta).abs() + bdelta) + bdelta + (d + 4) * e * (g.abs() @ x.abs().t() + delta.abs()))
            bds += eta * (1 + (dp - delta).abs() + bdelta)
            out["dq"][0][w, h] = ds @ b * c
            t = (bds + n * e * (ds.abs() + bds)) @ b.abs() * c
            out["dq"][1][w, h] = t + uo * (out["dq"][0][w, h].abs() + t)
            terms = n * grp
            out["dk"][0][w, h // grp] += ds.t() @ a * c
            out["dk"][1][w, h // grp] += (bds + terms * e * (ds.abs() + bds)).t() @ a.abs() * c
            out["dv"][0][w, h // grp] += p.t() @ g
            out["dv"][1][w, h // grp] += (p * (ep + u16 + terms * e) + eta).t() @ g.abs()
    for name in ("dk", "dv"):
        val, bound = out[name]
        out[name] = (val, bound + uo * (val.abs() + bound))
    return out


def _tiny(dtype):
    # Below the smallest normal number steps no longer shrink.
    return float(torch.finfo(dtype).tiny)


def _check(got, want, dtype, tokens):
    for name, t in got.items():
        val, bound = want[name]
        err = (t.double() - val)[:tokens].abs()
        over = err - bound[:tokens] - _tiny(dtype)
        assert torch.isfinite(t[:tokens]).all(), name
        if over.numel():
            assert float(over.max()) <= 0, f"{name}: {float(over.max()):.3e} over the bound, error {float(err.max()):.3e}"


def _run(q, k, v, do, plan, causal):
    o, lse = ct.flash_attn_packed_fwd(q, k, v, plan, causal=causal)
    dq, dk, dv = ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, causal=causal)
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)


LENS = [1, 0, 33, 64, 65, 127, 2, 129, 200]
MANY = [120, 65, 128, 1, 100, 33, 127, 129] * 9  # enough of like lengths that larger tiles are taken


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 1), (6, 2), (7, 1)])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_against_64_bits(dtype, d, hq, hkv, causal):
    x = _inputs(LENS, hq, hkv, d, dtype, seed=d + hq)
    plan = ct.packed_plan(LENS, hq, hkv)
    _check(_run(*x, plan, causal), _reference(*x, LENS, causal), dtype, plan.tokens)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_many_sequences(dtype, d, causal):
    x = _inputs(MANY, 12, 4, d, dtype, seed=d)
    plan = ct.packed_plan(MANY, 12, 4)
    _check(_run(*x, plan, causal), _reference(*x, MANY, causal), dtype, plan.tokens)


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 72), (torch.float32, 40), (torch.float16, 24), (torch.float32, 104)])
def test_many_sequences_between_the_tile_widths(dtype, d):
    x = _inputs(MANY, 8, 8, d, dtype, seed=d)
    plan = ct.packed_plan(MANY, 8, 8)
    _check(_run(*x, plan, True), _reference(*x, MANY, True), dtype, plan.tokens)


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 8), (torch.bfloat16, 40), (torch.float16, 80), (torch.bfloat16, 96),
                                     (torch.bfloat16, 120), (torch.float32, 4), (torch.float32, 44), (torch.float32, 100)])
def test_head_dims_between_the_tile_widths(dtype, d):
    x = _inputs(LENS, 4, 2, d, dtype, seed=d)
    plan = ct.packed_plan(LENS, 4, 2)
    _check(_run(*x, plan, True), _reference(*x, LENS, True), dtype, plan.tokens)


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 33), (torch.float16, 200), (torch.float32, 1), (torch.float32, 256),
                                     (torch.float64, 64), (torch.float64, 7)])
@pytest.mark.parametrize("causal", [True, False])
def test_generic_kernels(dtype, d, causal):
    lens = [1, 70, 0, 65]
    x = _inputs(lens, 6, 2, d, dtype, seed=d)
    plan = ct.packed_plan(lens, 6, 2)
    _check(_run(*x, plan, causal), _reference(*x, lens, causal), dtype, plan.tokens)


@gpu
def test_generic_policy_and_many_heads():
    lens = [100, 31]
    x = _inputs(lens, 130, 1, 32, torch.bfloat16)  # 130 query heads on one
    plan = ct.packed_plan(lens, 130, 1)
    want = _reference(*x, lens, True)
    _check(_run(*x, plan, True), want, torch.bfloat16, plan.tokens)
    x = _inputs(lens, 128, 1, 32, torch.bfloat16)
    plan = ct.packed_plan(lens, 128, 1)
    want = _reference(*x, lens, True)
    _check(_run(*x, plan, True), want, torch.bfloat16, plan.tokens)
    prev = ct.set_policy(ct.POLICY_GENERIC)
    try:
        _check(_run(*x, plan, True), want, torch.bfloat16, plan.tokens)
    finally:
        ct.set_policy(prev)


@gpu
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [2048], [1500, 3, 700], list(range(1, 40))])
def test_lengths(lens):
    x = _inputs(lens, 4, 2, 64, torch.bfloat16, seed=len(lens))
    plan = ct.packed_plan(lens, 4, 2)
    _check(_run(*x, plan, True), _reference(*x, lens, True), torch.bfloat16, plan.tokens)


@gpu
def test_empty_batches():
    for lens in ([], [0], [0, 0]):
        plan = ct.packed_plan(lens, 4, 2)
        q, k, v, do = _inputs([], 4, 2, 64, torch.bfloat16)
        r = _run(q, k, v, do, plan, True)
        assert r["o"].shape == (0, 4, 64) and r["lse"].shape == (0, 4)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_growing_scores(dtype):
    """Later keys score ever higher: the running maximum rises in every block."""
    lens, d = [500, 77], 64
    q, k, v, do = _inputs(lens, 4, 2, d, dtype)
    ramp = torch.cat([torch.linspace(0, 1, n) for n in lens]).cuda()[:, None, None]
    q = (q.float() + 3).to(dtype)
    k = (k.float() + 6 * ramp).to(dtype)
    plan = ct.packed_plan(lens, 4, 2)
    for causal in (True, False):
        _check(_run(q, k, v, do, plan, causal), _reference(q, k, v, do, lens, causal), dtype, plan.tokens)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_one_projection(dtype):
    """q, k, v as slices of one [tokens, (Hq + 2 Hkv) d] buffer, the gradients into slices of another; and
    [heads, tokens, d] storage seen as [tokens, heads, d]."""
    lens, hq, hkv, d = [65, 130, 1], 4, 2, 64
    x = _inputs(lens, hq, hkv, d, dtype)
    want = _reference(*x, lens, True)
    n = sum(lens)
    plan = ct.packed_plan(lens, hq, hkv)
    split = lambda b: [b[:, s].view(n, -1, d) for s in (slice(0, hq * d), slice(hq * d, (hq + hkv) * d), slice((hq + hkv) * d, None))]  # noqa: E731
    qkv = torch.cat([t.reshape(n, -1) for t in x[:3]], 1)
    grads = torch.full_like(qkv, 7.0)
    q, k, v = split(qkv)
    dq, dk, dv = split(grads)
    o, lse = ct.flash_attn_packed_fwd(q, k, v, plan, causal=True)
    ct.flash_attn_packed_bwd(q, k, v, o, x[3], lse, plan, causal=True, dq=dq, dk=dk, dv=dv)
    _check(dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv), want, dtype, n)
    y = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in x]
    o = torch.empty_like(y[0])
    assert o.stride() == y[0].stride()
    ct.flash_attn_packed_fwd(*y[:3], plan, causal=True, out=o, lse=lse)
    dq, dk, dv = ct.flash_attn_packed_bwd(*y[:3], o, y[3], lse, plan, causal=True)
    _check(dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv), want, dtype, n)


@gpu
def test_off_16_bytes_and_autograd():
    lens, hq, hkv, d = [40, 9], 4, 2, 32
    x = _inputs(lens, hq, hkv, d, torch.bfloat16)
    want = _reference(*x, lens, True)
    plan = ct.packed_plan(lens, hq, hkv)
    off = []
    for t in x:
        b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        b[1:] = t.reshape(-1)
        off.append(b[1:].view(t.shape))
    _check(_run(*off, plan, True), want, torch.bfloat16, plan.tokens)
    q, k, v = (t.detach().requires_grad_() for t in off[:3])
    o = ct.flash_attention_packed(q, k, v, plan, causal=True)
    o.backward(off[3])
    _check(dict(o=o.detach(), dq=q.grad, dk=k.grad, dv=v.grad), want, torch.bfloat16, plan.tokens)


@gpu
def test_gradient_by_differences():
    lens = [5, 1, 12]
    plan = ct.packed_plan(lens, 4, 2)
    q, k, v, _ = (t.requires_grad_() for t in _inputs(lens, 4, 2, 6, torch.float64))
    for causal in (True, False):
        assert torch.autograd.gradcheck(lambda a, b, c: ct.flash_attention_packed(a, b, c, plan, causal), (q, k, v))  # noqa: B023


@gpu
def test_rows_behind_the_last_sequence_are_left():
    lens, extra = [70, 3], 11
    x = _inputs(lens, 4, 2, 64, torch.bfloat16, extra=extra)
    n = sum(lens)
    for t in x:
        t[n:] = math.nan  # read by nobody
    plan = ct.packed_plan(lens, 4, 2)
    outs = [torch.full_like(t, 5.0) for t in (x[0], x[0], x[1], x[2])]
    lse = torch.full(x[0].shape[:2], 5.0, device="cuda")
    ct.flash_attn_packed_fwd(*x[:3], plan, causal=True, out=outs[0], lse=lse)
    ct.flash_attn_packed_bwd(*x[:3], outs[0], x[3], lse, plan, causal=True, dq=outs[1], dk=outs[2], dv=outs[3])
    want = _reference(*(t[:n] for t in x), lens, True)
    for name, t in zip(("o", "dq", "dk", "dv", "lse"), outs + [lse]):
        assert bool((t[n:] == 5.0).all()), name
        _check({name: t[:n]}, want, torch.bfloat16, n)


@gpu
def test_nan_and_infinity_stay_in_their_sequence():
    lens = [70, 90, 33]
    x = _inputs(lens, 4, 2, 64, torch.bfloat16)
    plan = ct.packed_plan(lens, 4, 2)
    clean = _run(*x, plan, True)
    bad = [t.clone() for t in x]
    for t, value in zip(bad, (math.nan, math.inf, math.nan, -math.inf)):
        t[75:120:7] = value  # inside the second sequence
    got = _run(*bad, plan, True)
    for name in clean:
        assert torch.equal(got[name][:70], clean[name][:70]) and torch.equal(got[name][160:], clean[name][160:]), name
    # A NaN in one query row alone is that row's alone in O.
    one = [t.clone() for t in x]
    one[0][100, 1] = math.nan
    o = ct.flash_attn_packed_fwd(*one[:3], plan, causal=True)[0]
    assert bool(o[100, 1].isnan().all())
    keep = torch.ones(o.shape[:2], dtype=torch.bool, device="cuda")
    keep[100, 1] = False
    assert torch.equal(o[keep], clean["o"][keep])


@gpu
def test_same_bits_every_time():
    lens = [300, 41, 200]
    for dtype in (torch.bfloat16, torch.float32):
        x = _inputs(lens, 6, 2, 64, dtype)
        plan = ct.packed_plan(lens, 6, 2)
        a, b = _run(*x, plan, True), _run(*x, plan, True)
        assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
def test_streams_and_graph():
    lens = [130, 64, 7]
    x = _inputs(lens, 4, 2, 64, torch.bfloat16)
    plan = ct.packed_plan(lens, 4, 2)
    want = _run(*x, plan, True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _run(*x, plan, True)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    o, lse = ct.flash_attn_packed_fwd(*x[:3], plan, causal=True, stream=side)
    side.synchronize()
    assert torch.equal(o, want["o"]) and torch.equal(lse, want["lse"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(*x, plan, True)
    for seed in range(3):
        for t, y in zip(x, _inputs(lens, 4, 2, 64, torch.bfloat16, seed=seed)):
            t.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(*x, plan, True)
        assert all(torch.equal(out[n], eager[n]) for n in out)


@gpu
def test_strides_of_single_heads_and_rows():
    """One head, or one token: that dimension's stride may be anything."""
    lens, d = [70, 5], 64
    x = _inputs(lens, 2, 1, d, torch.bfloat16)
    plan = ct.packed_plan(lens, 2, 1)
    want = _run(*x, plan, True)
    k, v = (t[:, 0].as_strided((75, 1, d), (d, 3, 1)) for t in x[1:3])
    got = _run(x[0], k, v, x[3], plan, True)
    assert all(torch.equal(got[n], want[n]) for n in want)
    one = ct.packed_plan([1], 2, 1)
    y = [t[:1] for t in x]
    odd = [t.as_strided(t.shape, (7, t.stride(1), 1)) for t in y]
    a, b = _run(*y, one, True), _run(*odd, one, True)
    assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
def test_offsets_past_32_bits():
    """Rows 2 MiB apart: the later ones of 4200 lie past 2^32 bytes and 2^32 elements."""
    lens, hq, hkv, d = [4100, 100], 2, 1, 64
    n = sum(lens)
    x = _inputs(lens, hq, hkv, d, torch.bfloat16)
    plan = ct.packed_plan(lens, hq, hkv)
    want = _run(*x, plan, True)
    buf = torch.empty((n, 1 << 20), dtype=torch.bfloat16, device="cuda")
    parts, at = [], 0
    for heads in (hq, hkv, hkv, hq, hq, hq, hkv, hkv):  # q k v do o dq dk dv
        parts.append(buf[:, at:at + heads * d].view(n, heads, d))
        at += heads * d
    for t, y in zip(parts, x):
        t.copy_(y)
    q, k, v, do, o, dq, dk, dv = parts
    _, lse = ct.flash_attn_packed_fwd(q, k, v, plan, causal=True, out=o)
    ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, causal=True, dq=dq, dk=dk, dv=dv)
    got = dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)
    assert all(torch.equal(got[name], want[name]) for name in want)


@gpu
def test_two_streams_at_once():
    lens = [400, 130, 64]
    plan = ct.packed_plan(lens, 8, 2)
    xs = [_inputs(lens, 8, 2, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [_run(*x, plan, True) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(_run(*x, plan, True))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(g[n], w[n]) for n in w)


@gpu
def test_binding_refusals():
    lens = [8, 4]
    plan = ct.packed_plan(lens, 4, 2)
    q, k, v, do = _inputs(lens, 4, 2, 64, torch.bfloat16)
    o, lse = ct.flash_attn_packed_fwd(q, k, v, plan)
    bad = [lambda: ct.flash_attn_packed_fwd(q[:11], k[:11], v[:11], plan),
           lambda: ct.flash_attn_packed_fwd(q[:, :2], k, v, plan),
           lambda: ct.flash_attn_packed_fwd(q, k, v[:, :1], plan),
           lambda: ct.flash_attn_packed_fwd(q, k.float(), v, plan),
           lambda: ct.flash_attn_packed_fwd(q, k, v.cpu(), plan),
           lambda: ct.flash_attn_packed_fwd(q.transpose(1, 2), k, v, plan),
           lambda: ct.flash_attn_packed_fwd(q.int(), k.int(), v.int(), plan),
           lambda: ct.flash_attn_packed_fwd(q, k, v, lens),
           lambda: ct.flash_attn_packed_fwd(q, k, v, plan, lse=lse.double()),
           lambda: ct.flash_attn_packed_fwd(q, k, v, plan, out=o[:, :, :32]),
           lambda: ct.flash_attn_packed_bwd(q, k, v, o, do, lse.t(), plan),
           lambda: ct.flash_attn_packed_bwd(q, k, v, o, do[:, :2], lse, plan),
           lambda: ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, dk=q),
           lambda: ct.packed_bwd_workspace_bytes(torch.bfloat16, plan, 4, 4, 64)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    with pytest.raises(RuntimeError, match="workspace"):
        ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="overlap"):
        ct.flash_attn_packed_fwd(q, k, v, plan, out=q.new_empty(64).expand(12, 4, 64))
    # Outputs on an input's memory, or on each other's.
    with pytest.raises(RuntimeError, match="input's memory"):
        ct.flash_attn_packed_fwd(q, k, v, plan, out=q)
    with pytest.raises(RuntimeError, match="input's memory"):
        ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, dq=q)
    with pytest.raises(RuntimeError, match="input's memory"):
        ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, dv=v)
    both = torch.empty_like(k)
    with pytest.raises(RuntimeError, match="share memory"):
        ct.flash_attn_packed_bwd(q, k, v, o, do, lse, plan, dk=both, dv=both)
    buf = q.new_empty((12, 8, 64))
    buf[:, :4] = q
    a, b = buf[:, :4], buf[:, 4:]  # apart within every row
    assert torch.equal(ct.flash_attn_packed_fwd(a, k, v, plan, out=b)[0], o)
    with pytest.raises(RuntimeError, match="input's memory"):
        ct.flash_attn_packed_fwd(a, k, v, plan, out=buf[:, 3:7])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            ct.packed_plan([4], 4, 2)
        q.mul_(1.0)  # a graph with nothing in it is not one
