"""The scaled lookup and the gradient by sorted tokens against sums in 64 bits.

Bounds: the lookup rounds one product once (the product in fp32, 2^-24, then half a step of the type); a
sum of n terms in fp32 is off by n 2^-24 of the terms' absolute sum, times the scale, then rounded once.
"""
import ctypes
import math

import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def _e(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def _expected(ids, dout, vocab, scale, before=None):
    """(value, bound) of the gradient."""
    flat, x = ids.reshape(-1).long(), dout.double().reshape(-1, dout.shape[-1])
    keep = (flat >= 0) & (flat < vocab)
    total, size = (torch.zeros((vocab, x.shape[1]), dtype=torch.float64, device=x.device) for _ in range(2))
    total.index_add_(0, flat[keep], x[keep])
    size.index_add_(0, flat[keep], x[keep].abs())
    count = torch.bincount(flat[keep], minlength=vocab)[:, None]
    value = total * scale
    bound = (count + 3) * _e(dout.dtype) * abs(scale) * size
    if before is not None:
        value = value + before.double()
        bound = bound + _e(dout.dtype) * value.abs()
    half = torch.finfo(dout.dtype).eps / 2
    return value, bound + half * (value.abs() + bound) + float(torch.finfo(dout.dtype).tiny)


def _check(got, want):
    value, bound = want
    over = (got.double() - value).abs() - bound
    assert torch.isfinite(got).all() and float(over.max()) <= 0, f"{float(over.max()):.3e} over the bound"


def _case(n, vocab, d, dtype, seed=0, spread=1.0, id_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    # spread 0: one id; 1: uniform; above: few ids many times.
    u = torch.rand(n, generator=g, dtype=torch.float64)
    ids = (u ** max(spread, 1.0) * vocab).long().clamp_(max=vocab - 1) if spread > 0 else torch.full((n,), vocab // 2)
    return ids.to(id_dtype).cuda(), torch.randn((n, d), generator=g).to(dtype).cuda()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 8, 33, 64, 100, 513, 768])
@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
def test_lookup(dtype, d, id_dtype):
    vocab = 97
    ids, _ = _case(211, vocab, 1, dtype, id_dtype=id_dtype)
    ids[5], ids[60], ids[210] = -1, vocab, 2 ** 31 - 1
    table = torch.randn((vocab, d), generator=torch.Generator().manual_seed(d)).to(dtype).cuda()
    scale = math.sqrt(d) + 0.3
    out = ct.embedding_lookup(ids, table, scale=scale)
    keep = (ids >= 0) & (ids < vocab)
    want = table[torch.where(keep, ids, 0).long()].double() * scale * keep[:, None]
    half = torch.finfo(dtype).eps / 2
    bound = want.abs() * (half + 3 * _e(dtype)) + float(torch.finfo(dtype).tiny)
    assert float(((out.double() - want).abs() - bound).max()) <= 0
    assert bool((out[~keep] == 0).all())
    plain = ct.embedding_lookup(ids.view(1, -1)[:, :210].contiguous(), table)
    assert plain.shape == (1, 210, d) and torch.equal(plain[0][keep[:210]], table[ids[:210][keep[:210]].long()])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,d,spread", [
    (1, 1, 1, 1), (1, 70000, 33, 1), (31, 5, 8, 1), (32, 40, 64, 1), (33, 2, 100, 1), (64, 64, 513, 2), (65, 1000, 768, 1),
    (1000, 511, 40, 1), (1000, 512, 40, 2), (4096, 65, 384, 1), (4096, 262143, 16, 1), (4097, 300, 24, 3), (5000, 50257, 72, 6),
    (5000, 300000, 7, 2), (9000, 3, 130, 1), (20000, 9, 12, 0), (70000, 1000, 20, 8)])
def test_gradient(dtype, n, vocab, d, spread):
    ids, dout = _case(n, vocab, d, dtype, seed=n, spread=spread)
    _check(ct.embedding_grad(ids, dout, vocab, scale=1.7), _expected(ids, dout, vocab, 1.7))


@gpu
@pytest.mark.parametrize("n", [40, 3000, 12000])
@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
def test_ids_outside_the_table(n, id_dtype):
    ids, dout = _case(n, 100, 48, torch.float32, id_dtype=id_dtype, spread=2)
    ids[::3] = -1
    ids[1::7] = 100
    ids[2::11] = 2 ** 31 - 1
    if id_dtype == torch.int64:
        ids[3::13] = 2 ** 32 + 5
    dout[ids < 0] = math.nan  # belongs to no row
    want = _expected(ids, dout, 100, 1.0)
    _check(ct.embedding_grad(ids, dout, 100), want)
    ids.fill_(-1)
    assert bool((ct.embedding_grad(ids, dout, 100) == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [0, 100, 6000])
def test_accumulate(dtype, n):
    ids, dout = _case(n, 70, 96, dtype, spread=2)
    before = torch.randn((70, 96), generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    got = ct.embedding_grad(ids, dout, 70, scale=0.5, out=before.clone(), accumulate=True)
    _check(got, _expected(ids, dout, 70, 0.5, before))
    untouched = torch.ones(70, dtype=torch.bool, device="cuda")
    untouched[ids.long()] = False
    assert torch.equal(got[untouched], before[untouched])
    stale = torch.full_like(before, math.nan)
    _check(ct.embedding_grad(ids, dout, 70, scale=0.5, out=stale), _expected(ids, dout, 70, 0.5))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_off_16_bytes(dtype):
    n, vocab, d = 700, 90, 64
    ids, dout = _case(n, vocab, d, dtype)
    big = torch.full((vocab * d + 9,), 3.0, dtype=dtype, device="cuda")
    x = torch.empty(n * d + 1, dtype=dtype, device="cuda")
    x[1:] = dout.reshape(-1)
    out = big[1:1 + vocab * d].view(vocab, d)
    _check(ct.embedding_grad(ids, x[1:].view(n, d), vocab, out=out), _expected(ids, dout, vocab, 1.0))
    assert float(big[0]) == 3.0 and bool((big[1 + vocab * d:] == 3.0).all())
    odd = torch.empty(vocab * d + 1, dtype=dtype, device="cuda")[1:].view(vocab, d)
    odd.copy_(dout[:vocab])
    assert torch.equal(ct.embedding_lookup(ids, odd), dout[:vocab][ids.long()])


@gpu
def test_same_bits_every_time_and_streams():
    ids, dout = _case(30000, 500, 40, torch.float32, spread=5)
    a = ct.embedding_grad(ids, dout, 500)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    b = ct.embedding_grad(ids, dout, 500, stream=side)
    side.synchronize()
    assert torch.equal(a, b)


@gpu
def test_graph():
    for n in (600, 9000):
        ids, dout = _case(n, 300, 64, torch.bfloat16)
        table = torch.randn((300, 64), device="cuda").bfloat16()
        ct.embedding_grad(ids, dout, 300)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ct.embedding_lookup(ids, table, 2.0)
            g = ct.embedding_grad(ids, dout, 300, 2.0)
        for seed in range(3):
            i2, d2 = _case(n, 300, 64, torch.bfloat16, seed=seed, spread=seed)
            ids.copy_(i2), dout.copy_(d2)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ct.embedding_lookup(ids, table, 2.0))
            assert torch.equal(g, ct.embedding_grad(ids, dout, 300, 2.0))


@gpu
def test_offsets_past_32_bits():
    """A table of 2.3e9 elements."""
    vocab, d = 70000, 33000
    ids = torch.tensor([69999, 3, 69999, 66000], dtype=torch.int32, device="cuda")
    dout = torch.randn((4, d), generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    grad = ct.embedding_grad(ids, dout, vocab)
    rows = torch.tensor([69999, 3, 66000], device="cuda")
    assert torch.equal(grad[rows[1:]], dout[[1, 3]])
    assert torch.equal(grad[69999], (dout[0].float() + dout[2].float()).bfloat16())
    assert torch.equal(ct.embedding_lookup(ids, grad), grad[ids.long()])
    grad[rows] = 0
    assert not any(bool(part.any()) for part in grad.split(7000))


@gpu
def test_two_streams_at_once():
    cases = [_case(n, 700, 64, torch.bfloat16, seed=n, spread=3) for n in (3000, 9000)]
    want = [ct.embedding_grad(i, x, 700) for i, x in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = [ct.embedding_grad(i, x, 700, stream=st) for (i, x), st in zip(cases, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@gpu
def test_autograd():
    ids = torch.randint(0, 9, (4, 6), device="cuda")
    table = torch.randn((9, 5), dtype=torch.float64, device="cuda", requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: ct.embedding(ids, t, 1.3), (table,))
    ct.embedding(ids, table, 1.3).sum().backward()  # a broadcast gradient
    want = _expected(ids, torch.ones((24, 5), dtype=torch.float64, device="cuda"), 9, 1.3)
    _check(table.grad, want)


@gpu
def test_autograd_takes_ids_and_a_table_of_any_order():
    ids = torch.randint(0, 9, (4, 6), device="cuda").t()
    leaf = torch.randn((5, 9), dtype=torch.float64, device="cuda", requires_grad=True)
    dout = torch.randn((5, 6, 4), dtype=torch.float64, device="cuda").permute(1, 2, 0)
    out = ct.embedding(ids, leaf.t(), 0.5)
    assert torch.equal(out, 0.5 * leaf.detach().t()[ids])  # a product by a power of two is exact
    out.backward(dout)
    _check(leaf.grad.t(), _expected(ids.reshape(-1), dout.reshape(24, 5), 9, 0.5))


@gpu
def test_binding_refusals():
    ids, dout = _case(10, 20, 8, torch.float32)
    table = torch.zeros((20, 8), device="cuda")
    for f in (lambda: ct.embedding_lookup(ids.float(), table), lambda: ct.embedding_lookup(ids.cpu(), table),
              lambda: ct.embedding_lookup(ids, table.t()), lambda: ct.embedding_lookup(ids, table.int()),
              lambda: ct.embedding_lookup(ids, table, out=table), lambda: ct.embedding_lookup(ids, table[0]),
              lambda: ct.embedding_grad(ids, dout[:9], 20), lambda: ct.embedding_grad(ids, dout, 0),
              lambda: ct.embedding_grad(ids, dout, 20, accumulate=True), lambda: ct.embedding_grad(ids, dout, 21, out=table),
              lambda: ct.embedding_grad(ids, dout, 20, out=table.half()),
              lambda: ct.embedding_grad(ids[::2], dout[::2], 20)):
        with pytest.raises(ValueError):
            f()
    square = torch.zeros((20, 8), device="cuda")
    with pytest.raises(RuntimeError, match="input's memory"):
        ct.embedding_lookup(torch.zeros(20, dtype=torch.int32, device="cuda"), square, out=square)
    with pytest.raises(RuntimeError, match="input's memory"):
        ct.embedding_grad(torch.zeros(20, dtype=torch.int32, device="cuda"), square, 20, out=square)
    with pytest.raises(RuntimeError, match="workspace"):
        ct.embedding_grad(ids, dout, 20, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_c_entry_refusals():
    lib = _capi.load()
    look = lambda dt=0, it=4, p=1 << 20, n=3, d=8, v=9: lib.ctattn_embedding_lookup(dt, it, p, p, p, 1.0, n, d, v, None)  # noqa: E731
    assert look() == 1 and "input's memory" in _capi.last_error()
    assert look(dt=4) == 1 and look(it=0) == 1 and look(p=None) == 1 and look(n=-1) == 1 and look(d=0) == 1 and look(v=0) == 1
    assert look(n=1 << 31) == 1 and look(v=(1 << 31) - 1) == 1 and look(d=1 << 30, n=1 << 30) == 1 and look(n=0, p=None) == 0
    need = lib.ctattn_embedding_grad_workspace_bytes(0, 3, 8, 9)
    assert need > 0 and lib.ctattn_embedding_grad_workspace_bytes(0, 3, 0, 9) == -1
    big = 1 << 20
    grad = lambda ws=256, size=need, p=big, n=3: lib.ctattn_embedding_grad(0, 4, p, 2 * big if p else p, 3 * big if p else p, 1.0, 0, ws,  # noqa: E731
                                                                           size, n, 8, 9, None)
    assert grad(ws=None) == 1 and grad(size=need - 1) == 1 and grad(ws=264) == 1 and grad(p=None) == 1
    assert ctypes.string_at(lib.ctattn_last_error()) != b""
