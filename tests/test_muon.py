"""Newton-Schulz orthogonalisation and the Muon step against 64 bits.

Single products are bounded element by element: one step with two of the three coefficients zero leaves
X, X X^T X or (X X^T)^2 X.  A factor is hi + lo, two fp16 numbers: off by 2^-22 (each of the two roundings by
half a step, 2^-11), and by 2^-25 / 256 where lo is subnormal; a product of two factors leaves lo lo out,
2^-22 again; fp32 sums of 3 K products are off by (3 K + 2) 2^-24 of their absolute sum.  Five steps amplify a rounding
by up to 3.4445^5, so there the error is held against that of the same iteration in fp32: factors of 2^-22
for its 2^-24 make it at most four times as large.
"""
import ctypes
import math

import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

gpu = pytest.mark.gpu
ABC = (3.4445, -4.7750, 2.0315)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _make(shape, dtype, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    *lead, m, n = shape
    k = max(1, min(m, n) // 4)
    x = torch.randn((*lead, m, k), generator=g) @ torch.randn((*lead, k, n), generator=g) / math.sqrt(k)
    return (size * (x + 0.5 * torch.randn(shape, generator=g))).to(dtype).cuda()


def _iterate(x, steps, abc, eps, dtype):
    """The definition, in `dtype`."""
    y = x.to(dtype)
    y = y / (y.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    if y.shape[-2] > y.shape[-1]:
        y = y.mT.contiguous()
    for _ in range(steps):
        gram = y @ y.mT.contiguous()
        y = abc[0] * y + (abc[1] * gram + abc[2] * (gram @ gram)) @ y
    return (y.mT if x.shape[-2] > x.shape[-1] else y).contiguous()


SHAPES = [(1, 1), (1, 70), (70, 1), (5, 3), (32, 32), (64, 129), (129, 64), (128, 128), (127, 200), (260, 131), (33, 1000)]


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_single_products(shape, dtype, which):
    x = _make((2, *shape), dtype, seed=sum(shape))
    abc = [0.0, 0.0, 0.0]
    abc[which] = 1.0
    got = ct.newton_schulz(x, steps=1, coeffs=abc)
    want = _iterate(x, 1, abc, 1e-7, torch.float64)
    y = x.double()
    y = y / (y.flatten(-2).norm(dim=-1)[..., None, None] + 1e-7)
    if shape[0] > shape[1]:
        y = y.mT
    r, c = y.shape[-2:]
    u, sub, e = 2.0 ** -22, 2.0 ** -33, 2.0 ** -24
    absy = y.abs() * (1 + 2 * e) + sub
    # (value of the factor, its absolute error) through the chain X -> A -> B -> B X.
    dy = absy * (u + 2 * e) + sub
    gram, ga = y @ y.mT, absy @ absy.mT
    dgram = (dy @ absy.mT) * 2 + ga * (u + (3 * c + 2) * e)
    dgram = dgram + (gram.abs() + dgram) * u + sub
    if which == 0:
        poly, dpoly = torch.eye(r, dtype=y.dtype, device=y.device).expand_as(gram), torch.zeros_like(gram)
    elif which == 1:
        poly, dpoly = gram, dgram + gram.abs() * e
    else:
        ab = gram.abs() + dgram
        poly, dpoly = gram @ gram, 2 * dgram @ ab + (ab @ ab) * (u + (3 * r + 4) * e)
    dpoly = dpoly + (poly.abs() + dpoly) * u + sub
    pa = poly.abs() + dpoly
    bound = dpoly @ absy + pa @ dy + (pa @ absy) * (u + (3 * r + 2) * e)
    if shape[0] > shape[1]:
        bound = bound.mT
    bound = bound + HALF[dtype] * (want.abs() + bound) + float(torch.finfo(dtype).tiny)
    over = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all() and float(over.max()) <= 0, f"{float(over.max()):.2e} over, error {float((got.double() - want).abs().max()):.2e}"


def _check_steps(got, x, steps=5, abc=ABC, eps=1e-7):
    want = _iterate(x, steps, abc, eps, torch.float64)
    plain = _iterate(x, steps, abc, eps, torch.float32).double()
    norm = lambda t: t.flatten(-2).norm(dim=-1)  # noqa: E731
    allowed = 4 * norm(plain - want) + (HALF[got.dtype] + 2.0 ** -22) * norm(want)
    err = norm(got.double() - want)
    assert bool((err <= allowed).all()), f"errors {err.tolist()}, allowed {allowed.tolist()}"


@gpu
@pytest.mark.parametrize("shape", [(3, 64, 64), (2, 3, 100, 333), (24, 130, 128), (1, 384, 1536), (700, 300), (1000, 31), (520, 520)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_five_steps(shape, dtype):
    x = _make(shape, dtype, seed=len(shape))
    _check_steps(ct.newton_schulz(x), x)


@gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 12])
def test_other_steps_and_coefficients(steps):
    x = _make((2, 90, 140), torch.float32)
    abc = (1.875, -1.25, 0.375)  # converges without overshoot
    _check_steps(ct.newton_schulz(x, steps=steps, coeffs=abc, eps=1e-3), x, steps, abc, 1e-3)


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-7, 1e12, 1e30])
def test_magnitudes(size):
    x = _make((60, 80), torch.float32, size=size)
    eps = 1e-7 if size > 1e-6 else 0.0
    _check_steps(ct.newton_schulz(x, eps=eps), x.double() / size, eps=0.0 if size > 1 or eps == 0 else eps / size)


@gpu
def test_zeros_nan_and_in_place():
    x = _make((3, 40, 50), torch.float32)
    x[1] = 0
    clean = ct.newton_schulz(x)
    assert bool((clean[1] == 0).all()) and torch.isfinite(clean).all()
    bad = x.clone()
    bad[1, 3, 4] = math.nan
    got = ct.newton_schulz(bad)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2]) and bool(got[1].isnan().all())
    bad[1, 3, 4] = math.inf
    assert bool((~torch.isfinite(ct.newton_schulz(bad)[1])).any())
    y = x.clone()
    assert ct.newton_schulz(y, out=y) is y and torch.equal(y, clean)
    assert ct.newton_schulz(x[:0]).shape == (0, 40, 50)


@gpu
def test_same_bits_streams_and_graph():
    x = _make((4, 200, 150), torch.bfloat16)
    a = ct.newton_schulz(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    b = ct.newton_schulz(x, stream=side)
    side.synchronize()
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ct.newton_schulz(x)
    for seed in range(3):
        x.copy_(_make((4, 200, 150), torch.bfloat16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ct.newton_schulz(x))


@gpu
def test_two_streams_at_once():
    xs = [_make((3, 130, 200), torch.float32, seed=1), _make((700, 260), torch.float32, seed=2)]
    want = [ct.newton_schulz(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = [ct.newton_schulz(x, stream=st) for x, st in zip(xs, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@gpu
@pytest.mark.parametrize("shape", [(1024, 1024), (1100, 1300), (2, 1024, 2048)])
def test_large_tiles(shape):
    x = _make(shape, torch.float32, seed=shape[-1])
    _check_steps(ct.newton_schulz(x), x)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("count", [1, 5, 70])
def test_muon_update(dtype, nesterov, count):
    shapes = [(40, 24), (24, 40), (40, 24)] if count == 5 else [(33, 20)]
    shapes = [shapes[i % len(shapes)] for i in range(count)]
    params = [_make(s, dtype, seed=i) for i, s in enumerate(shapes)]
    moments = [_make(s, torch.float32, seed=100 + i) for i, s in enumerate(shapes)]
    grads = [_make(s, dtype, seed=200 + i) for i, s in enumerate(shapes)]
    lr, mu, wd = 0.03, 0.9, 0.1
    p0, m0 = [p.double() for p in params], [m.double() for m in moments]
    ct.muon_update(params, grads, moments, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd)
    for p, g, m, pw, mw in zip(params, grads, moments, p0, m0):
        want_m = mu * mw + g.double()
        # momentum rounds to fp32, the sum once.
        assert float(((m.double() - want_m).abs() - 2.0 ** -23 * (want_m.abs() + (mu * mw).abs())).max()) <= 0
        u = (g.float() + mu * m if nesterov else m).double()
        o = _iterate(u, 5, ABC, 1e-7, torch.float64)
        plain = _iterate(u.float(), 5, ABC, 1e-7, torch.float32).double()
        s = lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        want = (1 - lr * wd) * pw - s * o
        # Newton-Schulz as above; u itself is off by 2^-23, which five steps amplify by at most 3.4445^5 of |X| = 1.
        err = float((p.double() - want).norm())
        allowed = s * (4 * float((plain - o).norm()) + (2.0 ** -22) * (3.4445 ** 5 + float(o.norm())))
        allowed += (HALF[dtype] + 2.0 ** -22) * float(want.norm() + pw.norm() * 2.0 ** -10)
        assert err <= allowed, f"{err:.3e} of {allowed:.3e}"


@gpu
@pytest.mark.parametrize("kind,dtype", [("Float", torch.float32), ("BFloat", torch.bfloat16), ("Half", torch.float16)])
def test_native_optimizer(kind, dtype):
    """The C++ host's optimizer moves its matrices as muon_update does: the same kernels in the same batches."""
    from cudatransformer_amd import cuda_transformer as ctm

    tensor = getattr(ctm, f"{kind}Tensor")
    shapes = {"a": (40, 24), "b": (24, 40), "c": (40, 24)}
    p = {n: _make(s, dtype, seed=i) for i, (n, s) in enumerate(shapes.items())}
    g = {n: _make(s, dtype, seed=50 + i) for i, (n, s) in enumerate(shapes.items())}
    to = lambda t: tensor.fromNumpy(t.double().cpu().numpy())  # noqa: E731
    params, grads = {n: to(t) for n, t in p.items()}, {n: to(t) for n, t in g.items()}
    opt = getattr(ctm, f"{kind}MuonOptimizer")(params, lr=0.03, momentum=0.9, decay=0.1)
    moments = {n: torch.zeros(s, device="cuda") for n, s in shapes.items()}
    for _ in range(2):
        opt.step(grads)
        ct.muon_update([p[n] for n in p], [g[n] for n in p], [moments[n] for n in p], lr=0.03, momentum=0.9, weight_decay=0.1)
    for n in p:
        assert torch.equal(torch.from_numpy(params[n].numpy()).double(), p[n].double().cpu()), n
    with pytest.raises(ValueError):
        opt.step({"a": grads["a"]})
    with pytest.raises(ValueError):
        getattr(ctm, f"{kind}MuonOptimizer")({"v": tensor.fromNumpy(torch.zeros(5).numpy())})
    assert not hasattr(ctm, "DoubleMuonOptimizer")


@gpu
def test_state_of_16_bit_parameters_is_kept():
    p = torch.nn.Parameter(_make((12, 9), torch.bfloat16))
    p.grad = _make((12, 9), torch.bfloat16, seed=1)
    opt = ct.Muon([p])
    opt.step()
    saved = opt.state_dict()
    again = ct.Muon([p])
    again.load_state_dict(saved)
    got, want = again.state[p]["moment"], opt.state[p]["moment"]
    assert got.dtype == torch.float32 and torch.equal(got, want) and got.data_ptr() != want.data_ptr()
    again.step()


@gpu
def test_binding_refusals():
    x = _make((8, 6), torch.float32)
    for f in (lambda: ct.newton_schulz(x.double()), lambda: ct.newton_schulz(x.t()), lambda: ct.newton_schulz(x.cpu()),
              lambda: ct.newton_schulz(x[0]), lambda: ct.newton_schulz(x, out=x.half()), lambda: ct.newton_schulz(x, steps=0),
              lambda: ct.newton_schulz(x, steps=101), lambda: ct.newton_schulz(x, coeffs=(65, 0, 0)),
              lambda: ct.newton_schulz(x, coeffs=(math.nan, 0, 0)), lambda: ct.newton_schulz(x, eps=-1.0),
              lambda: ct.newton_schulz(x, workspace=torch.empty(64, dtype=torch.uint8, device="cuda")),
              lambda: ct.muon_update([x], [x.clone()], []), lambda: ct.muon_update([x], [x.clone()], [x.half()]),
              lambda: ct.muon_update([x], [x], [x.clone()]), lambda: ct.muon_update([x], [x.half()], [x.clone()]),
              lambda: ct.muon_update([x, x], [x.clone(), x.clone()], [x.clone(), x.clone()]),
              lambda: ct.muon_update([x[0]], [x[0].clone()], [x[0].clone()])):
        with pytest.raises(ValueError):
            f()
    ct.muon_update([], [], [])


def test_c_entry_refusals():
    lib = _capi.load()

    def ns(dt=0, p=64, ws=256, size=1 << 40, mats=1, rows=8, cols=6, steps=5, a=1.0, eps=0.0):
        return lib.ctattn_newton_schulz(dt, p, p, ws, size, mats, rows, cols, steps, a, 0.0, 0.0, eps, None)

    assert ns(dt=3) == 801 and ns(dt=4) == 1 and ns(p=None) == 1 and ns(ws=None) == 1 and ns(ws=64) == 1
    assert ns(mats=-1) == 1 and ns(rows=0) == 1 and ns(cols=0) == 1 and ns(rows=1 << 21) == 1 and ns(mats=0, p=None) == 0
    assert ns(steps=0) == 1 and ns(steps=101) == 1 and ns(a=100.0) == 1 and ns(a=math.nan) == 1 and ns(eps=-1.0) == 1
    need = lib.ctattn_newton_schulz_workspace_bytes(0, 1, 8, 6)
    assert need > 0 and ns(size=need - 1) == 1 and lib.ctattn_newton_schulz_workspace_bytes(0, 1, 0, 6) == -1
    need = lib.ctattn_muon_update_workspace_bytes(1, 100, 8, 6)
    # Batches of 64 and the rest.
    assert need == max(lib.ctattn_muon_update_workspace_bytes(1, n, 8, 6) for n in (64, 36)) > 0
    one, two, three = ((ctypes.c_void_p * 1)(i << 20) for i in (1, 2, 3))
    none = (ctypes.c_void_p * 1)(None)

    def muon(p=one, g=two, m=three, count=1, size=1 << 40):
        return lib.ctattn_muon_update_multi(1, count, p, g, m, 256, size, 8, 6, 0.1, 0.9, 1, 0.0, 1.0, 5, 1.0, 0.0, 0.0, 0.0, None)

    assert muon(p=None) == 1 and muon(g=none) == 1 and muon(m=none) == 1 and muon(size=64) == 1 and muon(count=-1) == 1
    assert muon(count=0, p=None) == 0
    near = (ctypes.c_void_p * 1)((1 << 20) + 8 * 6 * 2 - 1)  # the last byte of p
    for bad in (dict(g=one), dict(m=one), dict(m=two), dict(g=near), dict(m=near)):
        assert muon(**bad) == 1 and "shares memory" in _capi.last_error()
    twice = (ctypes.c_void_p * 2)(1 << 20, 1 << 20)
    pair = lambda k: (ctypes.c_void_p * 2)(k << 20, (k + 1) << 20)  # noqa: E731
    assert muon(p=twice, g=pair(4), m=pair(6), count=2) == 1 and "shares memory" in _capi.last_error()
