"""Attention of requests that share a prompt in a paged cache (cudatransformer_amd.paged) against 64 bits."""
import ctypes
import math
import re

import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

gpu = pytest.mark.gpu


class Batch:
    """Prompts, requests and a cache with NaN wherever no token lies."""

    def __init__(self, dtype, prompts, sizes, new, own, hq, hkv, d, page, layout="token", seed=0, one_row=False, extra=3):
        g = torch.Generator().manual_seed(seed)
        self.prompts, self.sizes, self.new, self.own = prompts, sizes, new, own
        self.hq, self.hkv, self.d, self.page, self.dtype = hq, hkv, d, page, dtype
        held = [-(-n // page) for n in prompts + own]
        total = sum(held) + extra
        order = torch.randperm(total, generator=g).int()
        shape = (total, page, hkv, d) if layout == "token" else (total, hkv, page, d)
        caches = [torch.full(shape, math.nan, dtype=torch.float64) for _ in range(2)]
        if layout == "head":
            caches = [c.transpose(1, 2) for c in caches]
        width = [max([1] + h) for h in (held[:len(prompts)], held[len(prompts):])]
        self.ptable = torch.full((len(prompts), width[0]), -1, dtype=torch.int32)
        self.table = torch.full((len(own), width[1]), -1, dtype=torch.int32)
        self.keys, at = [], 0
        for i, n in enumerate(prompts + own):
            pages = order[at:at + held[i]]
            at += held[i]
            row = self.ptable[i] if i < len(prompts) else self.table[i - len(prompts)]
            row[:held[i]] = pages
            kv = []
            for c in caches:
                x = torch.randn((n, hkv, d), generator=g, dtype=torch.float64).to(dtype).double()
                j = torch.arange(n)
                c[pages.long()[j // page], j % page] = x
                kv.append(x)
            self.keys.append(kv)
        self.k, self.v = (c.to(dtype).cuda() for c in caches)
        if layout == "head":
            self.k, self.v = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (self.k, self.v))
        self.starts = torch.tensor([0] + new).cumsum(0).int()
        self.q = torch.randn((sum(new), hq, d), generator=g, dtype=torch.float64).to(dtype)

    def call(self, **kw):
        dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        args = dict(starts=None if all(n == 1 for n in self.new) else self.starts.cuda())
        if self.prompts:
            args.update(prefix_table=self.ptable.cuda(), prefix_lens=dev(self.prompts),
                        group_starts=dev([0] + torch.tensor(self.sizes).cumsum(0).tolist()))
        args.update(kw)
        return ct.flash_attn_shared_prefix(args.pop("q", self.q.cuda()), self.k, self.v, self.table.cuda(), dev(self.own), **args)

    def reference(self):
        """O, LSE and a bound of O's error, in 64 bits on the CPU."""
        group, d = self.hq // self.hkv, self.d
        o = torch.zeros(self.q.shape, dtype=torch.float64)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64)
        tol = torch.zeros_like(o)
        tol_lse = torch.zeros_like(lse)
        half = torch.finfo(self.dtype).eps / 2
        group_of = [g for g, n in enumerate(self.sizes) for _ in range(n)]
        for i, n in enumerate(self.new):
            for t in range(n):
                row = int(self.starts[i]) + t
                seen = max(0, self.own[i] - n + t + 1)
                parts = [x[:seen] for x in self.keys[len(self.prompts) + i]]
                if i < len(group_of):
                    parts = [torch.cat([a, b]) for a, b in zip(self.keys[group_of[i]], parts)]
                k, v = (x.repeat_interleave(group, 1) for x in parts)
                if len(k) == 0:
                    continue
                s = torch.einsum("hd,khd->hk", self.q[row].double(), k) / math.sqrt(d)
                z = torch.logsumexp(s, 1)
                p = torch.exp(s - z[:, None])
                o[row], lse[row] = torch.einsum("hk,khd->hd", p, v), z
                # P and O are rounded by half a step each (P once more where it leaves an accumulator of 32 bits);
                # scores are sums of d products in 32 bits and enter an exponential, sums run over the keys.
                a = torch.einsum("hk,khd->hd", p, v.abs())
                big = 1 + torch.einsum("hd,khd->hk", self.q[row].double().abs(), k.abs()).amax(1) / math.sqrt(d)
                small = torch.finfo(torch.float64 if self.dtype == torch.float64 else torch.float32).eps / 2
                rel = small * (len(k) + 2 * (d + 8) * big + 64)
                tol[row] = half * (a + o[row].abs()) + rel[:, None] * a
                tol_lse[row] = rel + small * lse[row].abs()
        return o, lse, tol, tol_lse

    def check(self, got):
        o, lse, tol, tol_lse = self.reference()
        here, here_lse = got[0].double().cpu(), got[1].double().cpu()
        assert torch.isfinite(here).all()
        worst = ((here - o).abs() - tol).max()
        assert worst <= 0, f"O is {float(worst):.3g} past its bound"
        none = lse == -math.inf
        assert torch.equal(here_lse == -math.inf, none)
        assert ((here_lse - lse).abs()[~none] <= tol_lse[~none]).all()


F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
CASES = {
    # one token a request
    "decode-bf16": dict(dtype=BF16, prompts=[133], sizes=[5], new=[1] * 5, own=[1, 40, 16, 129, 300], hq=8, hkv=2, d=128, page=16),
    "decode-f32": dict(dtype=F32, prompts=[200], sizes=[4], new=[1] * 4, own=[56, 1, 17, 16], hq=6, hkv=6, d=64, page=16),
    "decode-f16-groups": dict(dtype=F16, prompts=[70, 1, 257], sizes=[2, 3, 1], new=[1] * 6, own=[3, 9, 33, 64, 65, 1], hq=4, hkv=4,
                              d=64, page=32, layout="head"),
    # many rows of one key head beside the prompt: tiles of 128, more than one
    "decode-many": dict(dtype=BF16, prompts=[700], sizes=[40], new=[1] * 40, own=list(range(1, 41)), hq=16, hkv=2, d=64, page=16),
    "decode-many-f32": dict(dtype=F32, prompts=[300, 40], sizes=[20, 19], new=[1] * 39, own=[7 * i % 90 + 1 for i in range(39)], hq=8,
                            hkv=2, d=128, page=8),
    # no prompt, an empty one, empty groups, requests without own tokens, requests outside the groups
    "no-prompt": dict(dtype=BF16, prompts=[], sizes=[], new=[1] * 3, own=[5, 130, 64], hq=4, hkv=2, d=64, page=16),
    "empty": dict(dtype=BF16, prompts=[0, 33, 12], sizes=[2, 0, 2], new=[1] * 4, own=[0, 7, 0, 20], hq=4, hkv=1, d=32, page=16),
    "empty-f32": dict(dtype=F32, prompts=[0, 33], sizes=[1, 1], new=[1] * 3, own=[0, 0, 0], hq=2, hkv=1, d=40, page=4),
    "outside": dict(dtype=F16, prompts=[90], sizes=[2], new=[1] * 4, own=[3, 4, 5, 6], hq=4, hkv=4, d=128, page=64),
    # several tokens a request, some none
    "several": dict(dtype=BF16, prompts=[150], sizes=[4], new=[5, 0, 37, 1], own=[5, 3, 70, 90], hq=8, hkv=2, d=64, page=16),
    "several-groups": dict(dtype=F32, prompts=[65, 64], sizes=[1, 3], new=[1, 2, 3, 33], own=[31, 2, 64, 40], hq=3, hkv=3, d=32, page=16),
    "several-tall": dict(dtype=F16, prompts=[300, 10], sizes=[3, 2], new=[150, 3, 61, 0, 130], own=[170, 3, 64, 10, 131], hq=8, hkv=4, d=128,
                         page=32, layout="head"),
    # head dims that fill part of a tile, pages of one token and pages beyond the batch
    "width-40": dict(dtype=BF16, prompts=[77], sizes=[3], new=[1] * 3, own=[50, 3, 17], hq=4, hkv=2, d=40, page=1),
    "width-80": dict(dtype=F16, prompts=[129], sizes=[3], new=[1, 4, 2], own=[50, 30, 17], hq=5, hkv=1, d=80, page=256),
    "width-96-many": dict(dtype=F32, prompts=[129], sizes=[30], new=[1] * 30, own=[20] * 30, hq=10, hkv=2, d=96, page=2, layout="head"),
    "width-24": dict(dtype=BF16, prompts=[40], sizes=[2], new=[1, 1], own=[5, 40], hq=7, hkv=1, d=24, page=16),
    # the generic kernel: other head dims, fp64
    "generic-33": dict(dtype=BF16, prompts=[30], sizes=[2], new=[1, 3], own=[5, 70], hq=2, hkv=1, d=33, page=8),
    "generic-200": dict(dtype=F32, prompts=[66], sizes=[2], new=[1, 1], own=[5, 1], hq=2, hkv=2, d=200, page=16),
    "generic-f64": dict(dtype=F64, prompts=[70, 0], sizes=[2, 1], new=[2, 1, 3], own=[65, 9, 2], hq=4, hkv=2, d=64, page=16),
}


@gpu
@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("policy", [_capi.POLICY_AUTO, _capi.POLICY_GENERIC])
def test_against_64_bits(name, policy):
    b = Batch(**CASES[name])
    old = ct.set_policy(policy)
    try:
        b.check(b.call())
    finally:
        ct.set_policy(old)


@gpu
def test_wide_groups():
    """More query heads than a tile has rows to one key head, and more than the MFMA kernels take."""
    for hq in (48, 128, 144):
        b = Batch(BF16, [90], [3], [1, 2, 1], [10, 33, 70], hq, 1, 64, 16)
        b.check(b.call())


@gpu
def test_many_splits():
    """Tables much wider than what they hold, so that most stretches of keys are empty."""
    b = Batch(BF16, [1000], [2], [1, 1], [3, 500], 4, 2, 64, 16)
    wide = torch.cat([b.ptable, torch.full((1, 4000), -1, dtype=torch.int32)], 1)
    b.table = torch.cat([b.table, torch.full((2, 3000), 7, dtype=torch.int32)], 1)
    b.ptable = wide
    b.check(b.call())


@gpu
def test_strides_and_given_outputs():
    """q and o as slices of wider rows, tables as slices, given outputs, and rows behind the last request left alone."""
    b = Batch(F16, [100], [3], [2, 1, 4], [20, 5, 64], 4, 2, 64, 16)
    rows = sum(b.new) + 5
    fused = torch.randn((rows, 8, 64)).half().cuda()
    fused[:rows - 5, 2:6] = b.q.cuda()
    out = torch.full((rows, 6, 64), 7.0, dtype=F16, device="cuda")
    lse = torch.full((rows, 4), 3.0, device="cuda")
    tables = [torch.cat([t, t.new_full((len(t), 3), -5)], 1).cuda() for t in (b.table, b.ptable)]
    got = ct.flash_attn_shared_prefix(fused[:, 2:6], b.k, b.v, tables[0][:, :-3], torch.tensor(b.own, dtype=torch.int32, device="cuda"),
                                      tables[1][:, :-3], torch.tensor(b.prompts, dtype=torch.int32, device="cuda"),
                                      starts=b.starts.cuda(), out=out[:, 1:5], lse=lse)
    assert got[1] is lse
    b.check((out[:rows - 5, 1:5], lse[:rows - 5]))
    assert (out[rows - 5:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 5] == 7).all() and (lse[rows - 5:] == 3).all()
    # Allocated here they are zeros, with nothing seen.
    o, z = b.call(q=fused[:, 2:6])
    b.check((o[:rows - 5], z[:rows - 5]))
    assert (o[rows - 5:] == 0).all() and (z[rows - 5:] == -math.inf).all()


@gpu
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 33)])
def test_numbers_out_of_range(dtype, d):
    """Pages outside the cache are read as page 0, lengths are cut to the tables, starts to the rows."""
    b = Batch(dtype, [64], [2], [1, 1], [40, 20], 2, 1, d, 16)
    b.k.nan_to_num_(0.5)
    b.v.nan_to_num_(0.5)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, ptable = b.table.cuda(), b.ptable.cuda()
    table[0, 1], ptable[0, 2] = 1 << 30, -7
    zero_t, zero_p = table.clone(), ptable.clone()
    zero_t[0, 1], zero_p[0, 2] = 0, 0
    table[1, 2:], zero_t[1, 2:] = -1, 0
    got = ct.flash_attn_shared_prefix(b.q.cuda(), b.k, b.v, table, dev([40, 1 << 30]), ptable, dev([2000000000]))
    want = ct.flash_attn_shared_prefix(b.q.cuda(), b.k, b.v, zero_t, dev([40, 48]), zero_p, dev([64]))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = ct.flash_attn_shared_prefix(b.q.cuda(), b.k, b.v, zero_t, dev([-3, 20]), zero_p, dev([-1]), starts=dev([-9, 1, 100]),
                                      group_starts=dev([-4, 77]))
    want = ct.flash_attn_shared_prefix(b.q.cuda(), b.k, b.v, zero_t, dev([0, 20]), zero_p, dev([0]), starts=dev([0, 1, 2]))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@gpu
def test_infinite_scores_of_one_request():
    """A request whose keys are not finite reaches no other one."""
    b = Batch(BF16, [50], [3], [1, 1, 1], [20, 33, 5], 4, 2, 64, 16)
    want = b.call()[0]
    b.k[b.table[1, 0].item()] = math.inf
    got = b.call()[0]
    assert torch.equal(got[[0, 2]], want[[0, 2]])


@gpu
def test_streams_graphs_and_workspaces():
    """Another stream, and captured calls that replay on other lengths, pages and prompts, each with its own workspace."""
    a = Batch(BF16, [120, 31], [2, 2], [1] * 4, [9, 64, 1, 70], 8, 2, 64, 16, seed=1)
    b = Batch(BF16, [60, 128], [2, 2], [1] * 4, [40, 3, 77, 5], 8, 2, 64, 16, seed=2, extra=9)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = max(a.k.shape[0], b.k.shape[0])
    k, v = (torch.zeros((pages, 16, 2, 64), dtype=BF16, device="cuda") for _ in range(2))
    q = torch.zeros((4, 8, 64), dtype=BF16, device="cuda")
    table, ptable = (torch.zeros((n, 8), dtype=torch.int32, device="cuda") for n in (4, 2))
    lens, plens = dev([0] * 4), dev([0] * 2)
    need = ct.shared_prefix_workspace_bytes(BF16, 4, 4, 2, 8, 2, 64, 16, 8, 8)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def fill(x):
        k[:x.k.shape[0]], v[:x.k.shape[0]] = x.k, x.v
        q.copy_(x.q)
        table[:, :x.table.shape[1]] = x.table.cuda()
        ptable[:, :x.ptable.shape[1]] = x.ptable.cuda()
        lens.copy_(dev(x.own))
        plens.copy_(dev(x.prompts))

    call = lambda **kw: ct.flash_attn_shared_prefix(q, k, v, table, lens, ptable, plens, **kw)  # noqa: E731
    fill(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(stream=side)
    side.synchronize()
    a.check(got)
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for kw in (dict(workspace=ws), dict()):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(**kw))
        graphs.append(g)
    for x in (a, b, a, b):
        fill(x)
        ws.fill_(255)
        for g, out in zip(graphs, outs):
            g.replay()
            call()
            torch.cuda.synchronize()
            x.check(out)


@gpu
def test_reproducible():
    b = Batch(BF16, [900], [30], [1] * 30, [11 * i % 200 for i in range(30)], 8, 2, 128, 16)
    first = b.call()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, b.call()))


@gpu
def test_past_32_bits():
    """Pages whose bytes lie beyond 2^32."""
    pages, page, h, d = 140000, 16, 8, 128
    k = torch.zeros((pages, page, h, d), dtype=BF16, device="cuda")
    assert pages * page * h * d * 2 > 1 << 32
    v = k  # read alone
    g = torch.Generator(device="cuda").manual_seed(3)
    for at in (pages - 1, pages - 2):
        k[at] = torch.randn((page, h, d), generator=g, device="cuda").to(BF16)
    q = torch.randn((2, h, d), generator=g, device="cuda").to(BF16)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    far = ct.flash_attn_shared_prefix(q, k, v, dev([[pages - 1]] * 2), dev([16, 3]), dev([[pages - 2]]), dev([16]))
    near = k[-2:].clone()
    want = ct.flash_attn_shared_prefix(q, near, near, dev([[1]] * 2), dev([16, 3]), dev([[0]]), dev([16]))
    assert all(torch.equal(x, y) for x, y in zip(far, want)) and float(want[0].float().abs().max()) > 0


@gpu
def test_refusals():
    b = Batch(BF16, [20], [2], [1, 1], [4, 5], 4, 2, 32, 16)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q, t, pt, n, pn = b.q.cuda(), b.table.cuda(), b.ptable.cuda(), dev(b.own), dev(b.prompts)
    f = ct.flash_attn_shared_prefix
    bad = [lambda: f(b.q, b.k, b.v, t, n, pt, pn), lambda: f(q[0], b.k, b.v, t, n, pt, pn), lambda: f(q.float(), b.k, b.v, t, n, pt, pn),
           lambda: f(q.int(), b.k, b.v, t, n, pt, pn), lambda: f(q[:, :3], b.k, b.v, t, n, pt, pn),
           lambda: f(q, b.k[:, :15], b.v[:, :15], t, n, pt, pn), lambda: f(q, b.k, b.v[:-1], t, n, pt, pn),
           lambda: f(q, b.k, b.v, t.long(), n, pt, pn), lambda: f(q, b.k, b.v, t[:1], n, pt, pn),
           lambda: f(q, b.k, b.v, t, n.long(), pt, pn), lambda: f(q, b.k, b.v, t, n, pt, None), lambda: f(q, b.k, b.v, t, n, pt, pn.cpu()),
           lambda: f(q, b.k, b.v, t, n, torch.cat([pt] * 3), dev([1, 2, 3])), lambda: f(q[:1], b.k, b.v, t, n, pt, pn),
           lambda: f(q, b.k, b.v, t, n, pt, pn, starts=dev([0, 2])), lambda: f(q, b.k, b.v, t, n, pt, pn, group_starts=dev([0, 1, 2])),
           lambda: f(q, b.k, b.v, t, n, pt, pn, out=q[:, :2]), lambda: f(q, b.k, b.v, t, n, pt, pn, lse=torch.empty((2, 3), device="cuda")),
           lambda: f(q.transpose(1, 2), b.k, b.v, t, n, pt, pn)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    small = torch.empty(8, dtype=torch.uint8, device="cuda")
    for kw in (dict(out=q), dict(workspace=small), dict(out=b.k[0, :4].view(2, 4, 32))):
        with pytest.raises(RuntimeError):
            f(q, b.k, b.v, t, n, pt, pn, **kw)


def test_c_refusals():
    """What the entry point refuses before it touches memory."""
    lib = _capi.load()
    good = dict(dtype=1, rows=2, requests=2, groups=1, hq=4, hkv=2, d=64, pages=9, page_size=16, table_width=4, prefix_width=4)
    strides = (256, 64, 256, 64, 2048, 128, 64, 2048, 128, 64, 4, 4)

    def call(strides=strides, q=1 << 20, o=1 << 22, ws=1 << 30, ws_bytes=1 << 28, starts=None, **kw):
        a = {**good, **kw}
        s = (ctypes.c_int64 * 12)(*strides)
        sizes = [a[x] for x in ("rows", "requests", "groups", "hq", "hkv", "d", "pages", "page_size", "table_width", "prefix_width")]
        return lib.ctattn_shared_prefix_fwd(a["dtype"], q, 1 << 24, 1 << 26, 1 << 13, 1 << 14, 1 << 15, 1 << 16, None, starts, o, None, ws,
                                            ws_bytes, s, *sizes, 0, None)

    assert call(rows=0) == 0
    for kw in (dict(dtype=7), dict(hq=3), dict(hkv=0), dict(d=257), dict(d=0), dict(page_size=24), dict(page_size=0), dict(rows=-1),
               dict(rows=1 << 40), dict(requests=-1), dict(groups=-1), dict(pages=-1), dict(table_width=1 << 40), dict(q=None), dict(o=None),
               dict(rows=3), dict(requests=3, rows=3, groups=2), dict(ws=None), dict(ws_bytes=100), dict(ws=(1 << 30) + 8), dict(o=1 << 20),
               dict(o=1 << 24), dict(ws=1 << 24), dict(strides=(256, -64) + strides[2:]), dict(strides=strides[:2] + (0, 64) + strides[4:]),
               dict(strides=strides[:4] + (1 << 60,) + strides[5:])):
        assert call(**kw) != 0, kw
        assert _capi.last_error()
    for kw in (dict(hq=3), dict(d=0), dict(page_size=3)):
        a = {**good, **kw}
        assert lib.ctattn_shared_prefix_workspace_bytes(*[a[x] for x in ("dtype", "rows", "requests", "groups", "hq", "hkv", "d",
                                                                         "page_size", "table_width", "prefix_width")]) == -1


def needed(starts, group_starts, dtype=1, rows=32, requests=256, groups=1, hq=32, hkv=8, d=128, pages=1 << 20, page=16, width=128,
           prefix_width=256):
    """(bytes that the workspace query says, bytes that the call itself asks for); the call is given none and never launches."""
    lib = _capi.load()
    head = hkv * d
    strides = (ctypes.c_int64 * 12)(hq * d, d, hq * d, d, page * head, head, d, page * head, head, d, width, prefix_width)
    p = [(i + 1) << 44 for i in range(11)]
    rc = lib.ctattn_shared_prefix_fwd(dtype, *p[:7], p[7] if group_starts else None, p[8] if starts else None, p[9], None, p[10], 0, strides,
                                      rows, requests, groups, hq, hkv, d, pages, page, width, prefix_width, 0, None)
    said = re.search(r"workspace too small \(0 bytes, (\d+) needed\)", _capi.last_error())
    assert rc != 0 and said, _capi.last_error()
    return lib.ctattn_shared_prefix_workspace_bytes(dtype, rows, requests, groups, hq, hkv, d, page, width, prefix_width), int(said[1])


SIZES = [dict(rows=n) for n in (1, 2, 31, 32, 33, 100, 192, 255, 257, 300, 1000, 5000)]
SIZES += [dict(rows=n, groups=8) for n in (1, 17, 64, 65, 250, 400)]
SIZES += [dict(rows=n, requests=64, hq=16, hkv=16, d=64) for n in (1, 32, 63, 65, 2000)]
SIZES += [dict(rows=4096, requests=16, width=1024, prefix_width=64), dict(rows=8192, requests=8, width=2048, prefix_width=64),
          dict(rows=1800, requests=24, hq=16, hkv=16, d=64, page=32, width=22, prefix_width=129, dtype=2),
          dict(rows=7, requests=9, hq=6, hkv=6, d=64, dtype=0), dict(rows=5, requests=3, groups=0, prefix_width=0)]


@pytest.mark.parametrize("kw", SIZES, ids=str)
def test_workspace_of_calls_with_starts(kw):
    """Requests without a new token, and with several: what the query says is what the call needs."""
    for group_starts in (False, True):
        query, need = needed(True, group_starts, **kw)
        assert query == need


@pytest.mark.parametrize("kw", [dict(rows=n, requests=n, groups=g, hq=hq, hkv=8) for n in (1, 4, 48, 256) for g in (1, 3, 4) for hq in (8, 32, 512)],
                         ids=str)
def test_workspace_suffices_for_one_row_a_request(kw):
    forms = [(True, True), (False, True)]
    if kw["requests"] % kw["groups"] == 0:  # equal groups
        forms += [(True, False), (False, False)]
    got = [needed(*f, **kw) for f in forms]
    assert got[0][0] == max(need for _, need in got)


@gpu
@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 32, 8, 128), (F32, 4, 4, 64)])
def test_most_requests_have_no_new_token(dtype, hq, hkv, d):
    """Fewer rows than requests, one group and several, a request's first token and a later one."""
    own = [3 * i % 50 + 1 for i in range(40)]
    for rows in ([3], [0, 39], [1, 2, 3, 20, 21]):
        new = [int(i in rows) + (2 if i == 20 and 20 in rows else 0) for i in range(40)]
        for prompts, sizes in (([300], [40]), ([300, 17, 0], [10, 25, 5])):
            b = Batch(dtype, prompts, sizes, new, [max(n, m) for n, m in zip(own, new)], hq, hkv, d, 16)
            b.check(b.call(**(dict(group_starts=None) if len(prompts) == 1 else {})))


@pytest.mark.parametrize("width", [2047, 2048, 2049, 2050, 4097, 6145, 8191, 100001])
def test_at_most_64_stretches(width):
    """Of one request's own keys: each leaves 32 heads of 128 fp32 numbers, a maximum and a sum."""
    query, need = needed(True, False, rows=1, requests=1, groups=0, prefix_width=0, width=width)
    assert query == need and need % (32 * (128 + 2) * 4) == 0 and need // (32 * (128 + 2) * 4) <= 64


@pytest.mark.parametrize("kw", [dict(rows=8192, requests=8, width=2048), dict(rows=8192, requests=1, width=2048), dict(rows=2048, requests=1, width=8192),
                                dict(rows=4096, requests=4096, width=2048), dict(rows=30000, requests=20, width=8192),
                                dict(rows=256, requests=256, width=2048), dict(rows=1800, requests=24, width=8192, prefix_width=9000)], ids=str)
def test_workspace_of_wide_tables(kw):
    """What the splits leave is bounded by the rows, not by the width of tables made for the longest request: 256 MB of
    partial O (a number in 32 heads of 128, with a maximum and a sum for each) or one split, and as much as the prompt's."""
    query, need = needed(True, False, **kw)
    one = kw["rows"] * 32 * (128 + 2) * 4
    prompt = 512 * 128 * (128 + 2) * 4  # 512 work items of 128 rows
    assert need <= query <= max((256 << 20) * 130 // 128, one) + max(prompt, one) + 1024


@gpu
def test_many_rows_on_wide_tables():
    """So many rows that the partial O, not 64 stretches, bounds the splits of wide tables: 21 of 1472 keys, which two requests
    pass, and 21 of which all but the first are empty."""
    new = [700, 1, 1500, 0, 800]
    b = Batch(BF16, [40], [5], new, [900, 70, 1500, 3, 2000], 16, 2, 64, 16)
    for width in (1900, 120000):
        b.table = torch.cat([b.table, torch.full((5, width - b.table.shape[1]), -1, dtype=torch.int32)], 1)
        b.check(b.call())


@gpu
@pytest.mark.parametrize("d", [64, 33])
def test_one_of_two_outputs_given(d):
    """A given one keeps its rows of no request, an allocated one has nothing seen there."""
    b = Batch(BF16, [40], [3], [2, 1, 4], [20, 5, 64], 4, 2, d, 16)
    rows = sum(b.new) + 6
    q = torch.zeros((rows, 4, d), dtype=BF16, device="cuda")
    q[:-6] = b.q.cuda()
    kinds = dict(out=((rows, 4, d), BF16), lse=((rows, 4), F32))
    for what, (shape, dtype) in kinds.items():
        given = torch.full(shape, 7.0, dtype=dtype, device="cuda")
        for other, kind in kinds.values():  # what the allocator may hand out holds 5
            torch.full(other, 5.0, dtype=kind, device="cuda")
        got = b.call(q=q, **{what: given})
        b.check((got[0][:-6], got[1][:-6]))
        assert got[what == "lse"] is given and (given[-6:] == 7).all()
        assert (got[0][-6:] == 0).all() if what == "lse" else (got[1][-6:] == -math.inf).all()
