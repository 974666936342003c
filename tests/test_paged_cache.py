"""Pages and places of a paged cache, and writes into it (cudatransformer_amd.paged)."""
import ctypes

import pytest
import torch

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

gpu = pytest.mark.gpu


def reserve(lens, new, table, free, counters, page, most, offsets=None):
    """page_reserve, a request after the other, on lists."""
    table, taken, given, ring = [list(r) for r in table], *counters, len(free)
    width = len(table[0]) if table else 0
    slots, positions, starts, after, row, dealt, whole = [-1] * most, [0] * most, [], [], 0, 0, True
    avail = min(max(given - taken, 0), ring)
    used = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        raw, n, m = n, max(n, 0), max(m, 0)
        starts.append(min(row, 2**31 - 1))
        held, pages = -(-n // page), -(-(n + m) // page)
        fits = pages <= width and row + m <= most
        need = pages - held if fits else 0
        ok = fits and (need == 0 or dealt + need <= avail)
        if ok:
            for j in range(need):
                table[i][held + j] = free[(taken + dealt + j) % ring]
            if need:
                used = dealt + need
            for t in range(m):
                p = n + t
                slots[row + t] = table[i][p // page] * page + p % page
                positions[row + t] = p + (offsets[i] if offsets else 0)
        after.append(n + m if ok else raw)
        dealt += need
        row += m
    return slots, positions, starts + [min(row, 2**31 - 1)], after, [taken + used, given], table


def release(done, lens, table, free, counters, page):
    free, taken, given, ring = list(free), *counters, len(free)
    room = min(max(ring - (given - taken), 0), ring)
    after, at, used = [], 0, 0
    for d, n, row in zip(done, lens, table):
        pages = min(-(-max(n, 0) // page), len(row)) if d else 0
        ok = d and at + pages <= room
        if ok:
            for j in range(pages):
                free[(given + at + j) % ring] = row[j]
            used = at + pages
        after.append(0 if ok else n)
        at += pages
    return after, [taken, given + used], free


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def batch(rng, requests, most_held, most_new, page, spare, width=None):
    lens = [int(rng.integers(0, most_held + 1)) for _ in range(requests)]
    new = [int(rng.integers(0, most_new + 1)) for _ in range(requests)]
    held = [-(-n // page) for n in lens]
    need = [-(-(n + m) // page) - h for n, m, h in zip(lens, new, held)]
    width = width or max([1] + [h + k for h, k in zip(held, need)])
    order = rng.permutation(sum(held) + sum(need) + 50)
    at, table = 0, []
    for h in held:
        table.append([int(x) for x in order[at:at + h]] + [-1] * (width - h))
        at += h
    free = max(1, sum(need) + spare)
    ring = free + int(rng.integers(0, 9))
    taken = int(rng.integers(0, 10**10))
    pages = [-7] * ring
    for j in range(free):
        pages[(taken + j) % ring] = int(order[(at + j) % len(order)])
    return lens, new, table, pages, [taken, taken + free]


def run_reserve(lens, new, table, free, counters, page, most, offsets=None, **kw):
    t = dev(table).reshape(len(lens), -1)
    out = ct.page_reserve(dev(lens).reshape(-1), dev(new).reshape(-1), t, dev(free), dev(counters, torch.int64), page, most,
                          offsets=None if offsets is None else dev(offsets), **kw)
    return [x.tolist() for x in out] + [t.tolist()], out


@gpu
@pytest.mark.parametrize("requests,held,new,page,spare", [
    (1, 0, 1, 16, 0), (1, 40, 3000, 16, 5), (3, 50, 1, 1, 0), (65, 100, 1, 16, 0), (256, 90, 1, 16, 3), (256, 30, 5, 8, 0),
    (257, 30, 5, 8, 0), (1000, 0, 70, 32, 0), (1500, 200, 9, 4, -700), (300, 20, 20, 16, -90), (700, 30, 1, 16, -5),
    (5000, 60, 2, 64, 0), (40, 5000, 900, 2, -500)])
def test_reserve(requests, held, new, page, spare):
    import numpy as np

    rng = np.random.default_rng(requests * 7 + held)
    case = batch(rng, requests, held, new, page, spare)
    offsets = [int(rng.integers(0, 9999)) for _ in range(requests)]
    total = sum(case[1])
    for most, off in ((total + 3, offsets), (max(0, total - new), None), (total // 2, offsets)):
        got, _ = run_reserve(*case, page, most, off)
        assert got == [*reserve(*case, page, most, off)]


@gpu
def test_reserve_at_the_edges():
    page = 16
    # A table too narrow for one request, one that needs no page behind one that finds none, numbers below zero.
    case = ([15, 0, 31, 5, -4, 16], [1, 40, 1, -3, 2, 1], [[3] + [-1], [-1, -1], [4, 5], [6, -1], [-1, -1], [8, -1]], [1, 2, 9], [5, 7])
    got, _ = run_reserve(*case, page, 60)
    assert got == [*reserve(*case, page, 60)]
    assert got[3] == [16, 0, 32, 5, 2, 17] and got[4] == [7, 7]
    empty = run_reserve(*case[:3], [1, 2, 9], [7, 7], page, 60)[0]
    assert empty == [*reserve(*case[:3], [1, 2, 9], [7, 7], page, 60)] and empty[3] == [16, 0, 32, 5, -4, 16]
    assert run_reserve(*case[:3], [], [0, 0], page, 60)[0] == [*reserve(*case[:3], [1], [0, 0], page, 60)]
    # Lengths whose sums pass 32 bits are served where they fit and do no harm where they do not.
    big = ([2**31 - 1, 3, 2**31 - 1], [2**31 - 1, 2, 2**31 - 1], [[1], [2], [3]], [4, 5], [0, 2])
    assert run_reserve(*big, page, 40)[0] == [*reserve(*big, page, 40)]
    # No request, no row.
    none = ct.page_reserve(dev([]), dev([]), torch.empty((0, 4), dtype=torch.int32, device="cuda"), dev([1]),
                           dev([3, 4], torch.int64), page, 5)
    assert [x.tolist() for x in none] == [[-1] * 5, [0] * 5, [0], [], [3, 4]]
    assert run_reserve(*case, page, 0)[0] == [*reserve(*case, page, 0)]


@gpu
@pytest.mark.parametrize("requests,held,page", [(1, 40, 16), (5, 0, 16), (65, 100, 1), (256, 300, 16), (257, 30, 8), (3000, 90, 32),
                                                (20, 9000, 2)])
def test_release(requests, held, page):
    import numpy as np

    rng = np.random.default_rng(requests + held)
    lens, _, table, _, _ = batch(rng, requests, held, 0, page, 0)
    done = [bool(rng.integers(0, 2)) for _ in range(requests)]
    pages = sum(-(-n // page) for n in lens)
    for room in (pages + 9, pages // 3):
        free, taken = [100 + i for i in range(room + 4)], int(rng.integers(0, 10**10))
        counters = [taken, taken + 4]
        ring = dev(free)
        out = ct.page_release(dev(done, torch.bool), dev(lens), dev(table), ring, dev(counters, torch.int64), page)
        assert [x.tolist() for x in out] + [ring.tolist()] == [*release(done, lens, table, free, counters, page)]


@gpu
def test_a_batch_lives():
    """Steps of admission, decoding and release: no page belongs to two requests, none is lost, and what is written is read back.
    Captured and replayed beside the same steps on lists."""
    import numpy as np

    page, n, width, pages, most = 4, 9, 6, 30, 24
    rng = np.random.default_rng(5)
    free, counters = ct.page_pool(pages)
    lens, new, done = (torch.zeros(n, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.bool))
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    k = torch.randn((most, 2, 8), device="cuda")
    caches = [torch.zeros((pages, page, 2, 8), device="cuda") for _ in range(2)]

    def step():
        after, count = ct.page_release(done, lens, table, free, counters, page)
        slots, positions, starts, after, count = ct.page_reserve(after, new, table, free, count, page, most)
        ct.cache_write(k, -k, *caches, slots)
        lens.copy_(after)
        counters.copy_(count)
        return slots, positions, starts

    step()  # of no tokens
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    state = ([0] * n, [[-1] * width for _ in range(n)], list(range(pages)), [0, pages])
    kept = {i: [] for i in range(n)}
    for _ in range(40):
        gone = [bool(rng.random() < 0.25) for _ in range(n)]
        add = [int(rng.integers(0, 5)) if rng.random() < 0.8 else 0 for _ in range(n)]
        new.copy_(dev(add))
        done.copy_(dev(gone, torch.bool))
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        lists, tab, ring, count = state
        after, count, ring = release(gone, lists, tab, ring, count, page)
        slots, positions, starts, lists, count, tab = reserve(after, add, tab, ring, count, page, most)
        state = (lists, tab, ring, count)
        assert [x.tolist() for x in outs] == [slots, positions, starts]
        assert (lens.tolist(), table.tolist(), counters.tolist()) == (lists, tab, count)
        for i in range(n):
            if gone[i]:
                kept[i] = []
            if lists[i] == after[i] + add[i]:
                kept[i] += [k[starts[i] + t].clone() for t in range(add[i])]
            held = tab[i][:-(-lists[i] // page)]
            assert len(kept[i]) == lists[i]
            for p, x in enumerate(kept[i]):
                for c, y in zip(caches, (x, -x)):
                    assert torch.equal(c[held[p // page], p % page], y)
        owned = [p for i in range(n) for p in tab[i][:-(-lists[i] // page)]]
        assert len(set(owned)) == len(owned) == pages - (count[1] - count[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("rows,hkv,d,page,layout", [(1, 1, 1, 1, "token"), (5, 3, 40, 16, "head"), (70, 2, 33, 4, "token"),
                                                    (300, 8, 128, 64, "head"), (300, 4, 64, 16, "apart")])
def test_write(dtype, rows, hkv, d, page, layout):
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    pages = rows // page + 2
    shape = {"token": (pages, page, hkv, d), "head": (pages, hkv, page, d), "apart": (2, pages, page, hkv, d)}[layout]
    make = lambda s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    if layout == "apart":  # slices of one buffer, odd in the middle
        caches = list(make((pages, 2, page, hkv, d)).unbind(1))
    else:
        caches = [make(shape) for _ in range(2)]
        if layout == "head":
            caches = [c.transpose(1, 2) for c in caches]
    kv = make((rows, 2 * hkv + 1, d))
    k, v = kv[:, :hkv], kv[:, hkv + 1:]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows]
    slots[rows // 2:rows // 2 + 2] = torch.tensor([-1, pages * page], device="cuda")[:len(slots[rows // 2:rows // 2 + 2])]
    slots[-1:] = torch.where(slots[-1:] >= 0, slots[-1:], -(1 << 62))
    want = [c.clone() for c in caches]
    for c, x in zip(want, (k, v)):
        for n, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                c[s // page, s % page] = x[n]
    ct.cache_write(k, v, *caches, slots)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


@gpu
def test_write_past_32_bits_and_on_a_stream():
    cache = torch.zeros((140000, 16, 8, 128), dtype=torch.bfloat16, device="cuda")
    k = torch.randn((2, 8, 128), device="cuda").to(torch.bfloat16)
    slots = torch.tensor([140000 * 16 - 1, 5], device="cuda")
    with pytest.raises(RuntimeError):
        ct.cache_write(cache[0, :2], k, cache, cache, slots)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    second = torch.zeros_like(cache)
    torch.cuda.synchronize()
    ct.cache_write(k, k, cache, second, slots, stream=side)
    side.synchronize()
    for c in (cache, second):
        assert torch.equal(c[-1, -1], k[0]) and torch.equal(c[0, 5], k[1]) and int((c != 0).sum()) == int((k != 0).sum())


@gpu
def test_refusals():
    lens, table, (free, counters) = dev([1, 2]), dev([[0, 1], [2, 3]]), ct.page_pool(9)
    f = lambda **kw: ct.page_reserve(**{**dict(lens=lens, new_lens=lens, table=table, free=free, counters=counters, page_size=16,  # noqa: E731
                                               max_tokens=8), **kw})
    r = lambda **kw: ct.page_release(**{**dict(done=lens > 0, lens=lens, table=table, free=free, counters=counters, page_size=16), **kw})  # noqa: E731
    k = torch.zeros((2, 3, 8), device="cuda")
    cache = torch.zeros((4, 16, 3, 8), device="cuda")
    w = lambda **kw: ct.cache_write(**{**dict(k=k, v=k, k_cache=cache, v_cache=cache, slots=dev([0, 1], torch.int64)), **kw})  # noqa: E731
    bad = [lambda: f(lens=lens.cpu()), lambda: f(lens=lens.long()), lambda: f(new_lens=lens[:1]), lambda: f(table=table.long()),
           lambda: f(table=table[:1]), lambda: f(table=table.t()), lambda: f(free=free[None]), lambda: f(counters=counters.int()),
           lambda: f(page_size=12), lambda: f(page_size=0), lambda: f(max_tokens=-1), lambda: f(offsets=lens.long()), lambda: f(out=(lens,)),
           lambda: f(out=(counters,) * 5), lambda: r(done=lens), lambda: r(done=(lens > 0)[:1]), lambda: r(lens=lens[:1]), lambda: r(page_size=5),
           lambda: r(out=(lens, lens)), lambda: w(k=k.cpu()), lambda: w(k=k[0]), lambda: w(v=k[:1]), lambda: w(k=k.int(), v=k.int()),
           lambda: w(k=k.half()), lambda: w(k_cache=cache[:, :, :2]), lambda: w(k_cache=cache.half()), lambda: w(slots=dev([0, 1])),
           lambda: w(slots=dev([0], torch.int64)), lambda: w(k_cache=cache[:, :12], v_cache=cache[:, :12]),
           lambda: w(k=k.transpose(1, 2).contiguous().transpose(1, 2))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    new5 = lambda: [torch.empty(8, dtype=torch.int64, device="cuda"), torch.empty(8, dtype=torch.int64, device="cuda"),  # noqa: E731
                    torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda"),
                    torch.empty(2, dtype=torch.int64, device="cuda")]
    f(out=new5())
    for i, t in ((3, lens), (4, counters), (1, 0)):  # in place, and two outputs in one
        out = new5()
        out[i] = out[t] if isinstance(t, int) else t
        with pytest.raises(RuntimeError):
            f(out=out)
    with pytest.raises(RuntimeError):
        r(out=(lens, torch.empty_like(counters)))


def test_c_refusals():
    """What the entry points refuse before they touch memory."""
    lib = _capi.load()
    p = [1 << (12 + i) for i in range(12)]

    def res(requests=4, row=4, width=4, places=9, page=16, most=8, null=None):
        a = [None if i == null else x for i, x in enumerate(p[:11])]
        return lib.ctattn_page_reserve(*a, requests, row, width, places, page, most, None)

    def rel(requests=4, row=4, width=4, places=9, page=16, null=None):
        a = [None if i == null else x for i, x in enumerate(p[:7])]
        return lib.ctattn_page_release(*a, requests, row, width, places, page, None)

    for call in (res, rel):
        for kw in (dict(requests=-1), dict(requests=1 << 40), dict(row=3), dict(width=-1), dict(width=1 << 30), dict(places=-1), dict(page=0),
                   dict(page=24), dict(page=1 << 21), dict(null=0), dict(null=3), dict(null=4)):
            assert call(**kw) != 0, kw
    for kw in (dict(most=-1), dict(most=1 << 40), dict(null=6), dict(null=8)):
        assert res(**kw) != 0, kw
    strides = (64, 32, 64, 32, 2048, 64, 32, 2048, 64, 32)

    def wr(dtype=0, strides=strides, rows=4, hkv=2, d=32, pages=4, page=16, null=None, k=1 << 12):
        a = [None if i == null else x for i, x in enumerate([k, 1 << 14, 1 << 20, 1 << 22, 1 << 24])]
        return lib.ctattn_cache_write(dtype, *a, (ctypes.c_int64 * 10)(*strides), rows, hkv, d, pages, page, None)

    assert wr(rows=0) == 0
    for kw in (dict(dtype=9), dict(rows=-1), dict(hkv=0), dict(d=0), dict(d=1 << 30), dict(pages=-1), dict(page=3), dict(null=0), dict(null=3),
               dict(null=4), dict(k=1 << 20), dict(strides=(-64,) + strides[1:]), dict(strides=strides[:4] + (1 << 60,) + strides[5:])):
        assert wr(**kw) != 0, kw
