"""Calls of the generating operators that the documentation allows and nothing else makes: many rows put off at once, two calls
at a time, batches without requests, random numbers out of range."""
import math

import numpy as np
import pytest
import torch

import cudatransformer_amd as ct
from tests.test_sampling import check, logits_of, reference
from tests.test_shared_prefix import BF16, F32, Batch

gpu = pytest.mark.gpu


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


@gpu
@pytest.mark.parametrize("how", [dict(p=0.9), dict(k=4000), dict(k=4000, p=0.5), dict(p=0.9, m=0.02)])
def test_more_rows_put_off_than_have_a_place(how):
    """Nuclei of thousands of tokens in 1100 rows, of which 1024 are worked on together."""
    x, u = logits_of(1100, 8300, torch.bfloat16, 7, spread=1.0, sure=-3.0)
    check(x, u, **how)


@gpu
@pytest.mark.parametrize("vocab", [60, 400, 3001, 40000])
@pytest.mark.parametrize("how", [dict(), dict(top_k=9), dict(top_p=0.9), dict(top_p=0.99, temperature=9.0), dict(min_p=0.2)])
def test_random_numbers_out_of_range_draw_what_is_kept(vocab, how):
    x, _ = logits_of(5, vocab, torch.float32, vocab)
    u = torch.tensor([1.0, math.nan, -3.0, 7.0, math.inf], device="cuda")
    tokens, logprobs = ct.sample_tokens(x, u, **how)
    for i in range(5):
        at = [reference(x[i].cpu().numpy(), v, how.get("temperature", 1.0), how.get("top_k", 0), how.get("top_p", 1.0), how.get("min_p", 0.0))[0]
              for v in (0.0, float(np.nextafter(np.float32(1), np.float32(0))))]
        assert at[0] <= tokens[i].item() <= at[1]
        if i in (1, 2):  # no number and negative ones count as 0
            assert tokens[i].item() == at[0]
    assert torch.isfinite(logprobs).all()


@gpu
def test_two_calls_at_a_time():
    """On two streams, with nothing between them that waits."""
    x, u = logits_of(40, 50257, torch.bfloat16, 3, sure=-2.0)
    b = [Batch(BF16, [300, 70], [9, 8], [1] * 17, [5 * i + s for i in range(17)], 8, 2, 64, 16, seed=s) for s in (1, 2)]
    want = [ct.sample_tokens(x, u, 1.0, 0, p) for p in (0.9, 0.5)], [y.call() for y in b]
    streams = [torch.cuda.Stream() for _ in range(2)]
    args = []
    for y in b:  # made before, so that the calls are all that the streams do
        args.append((y.q.cuda(), y.k, y.v, y.table.cuda(), dev(y.own), y.ptable.cuda(), dev(y.prompts), dev([0, 9, 17])))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            got[0].append((i, ct.sample_tokens(x, u, 1.0, 0, (0.9, 0.5)[i], stream=s)))
            got[1].append((i, ct.flash_attn_shared_prefix(*args[i], stream=s)))
    torch.cuda.synchronize()
    for kind in (0, 1):
        for i, out in got[kind]:
            assert all(torch.equal(a, c) for a, c in zip(out, want[kind][i]))


@gpu
@pytest.mark.parametrize("dtype,d", [(F32, 32), (torch.float64, 8)])
def test_no_requests_and_no_groups(dtype, d):
    k = torch.zeros((2, 16, 1, d), dtype=dtype, device="cuda")
    q = torch.ones((3, 2, d), dtype=dtype, device="cuda")
    empty, table = dev([]), torch.empty((0, 4), dtype=torch.int32, device="cuda")
    # Rows of no request: zeros, or as they were.
    o, lse = ct.flash_attn_shared_prefix(q, k, k, table, empty, starts=dev([0]))
    assert (o == 0).all() and (lse == -math.inf).all()
    out = torch.full_like(q, 5.0)
    ct.flash_attn_shared_prefix(q, k, k, table, empty, dev([[0]]), dev([7]), dev([0, 0]), dev([0]), out=out)
    assert (out == 5).all()
    # No row, no group, a cache without pages.
    assert ct.flash_attn_shared_prefix(q[:0], k, k, table, empty)[0].shape == (0, 2, d)
    o, lse = ct.flash_attn_shared_prefix(q, k, k, dev([[0]] * 3), dev([1, 2, 16]), torch.empty((0, 3), dtype=torch.int32, device="cuda"), empty)
    assert (o == 0).all() and torch.allclose(lse.double().exp(), torch.tensor([1.0, 2.0, 16.0], dtype=torch.float64, device="cuda")[:, None])
    o, lse = ct.flash_attn_shared_prefix(q, k[:0], k[:0], dev([[0]] * 3), dev([1, 2, 16]))
    assert (o == 0).all() and (lse == -math.inf).all()


@gpu
def test_equal_groups_need_no_starts():
    b = Batch(BF16, [130, 70, 1], [4, 4, 4], [1] * 12, list(range(1, 13)), 8, 2, 64, 16)
    b.check(b.call(group_starts=None))
    got, want = b.call(group_starts=None), b.call()
    assert (got[0].float() - want[0].float()).abs().max() <= 2**-7 * want[0].float().abs().max()  # other splits: one rounding each


@gpu
def test_one_page_twice():
    """Two requests with the same pages, and one page twice in a request's table."""
    b = Batch(F32, [33], [2], [1, 1], [40, 40], 2, 1, 64, 16)
    b.table[1] = b.table[0]
    b.keys[2] = b.keys[1]
    b.check(b.call())
    b.table[0, 1] = b.table[0, 0]
    for x in b.keys[1]:
        x[16:32] = x[:16].clone()
    b.keys[2] = [x.clone() for x in b.keys[2]]
    c = Batch(F32, [33], [2], [1, 1], [40, 40], 2, 1, 64, 16)
    b.keys[2] = c.keys[1]
    b.check(b.call())


@gpu
def test_reservation_of_many_tokens_by_few_requests():
    """More rows than a workgroup's window, most of one request, and offsets near the end of 32 bits."""
    free, counters = ct.page_pool(5000)
    table = torch.full((3, 2048), -1, dtype=torch.int32, device="cuda")
    slots, positions, starts, lens, after = ct.page_reserve(dev([0, 5, 0]), dev([3, 30000, 2]), table, free, counters, 16, 30010,
                                                            offsets=dev([2**31 - 1, 7, -4]))
    assert starts.tolist() == [0, 3, 30003, 30005] and lens.tolist() == [3, 30005, 2] and after.tolist() == [1 + 1875 + 1, 5000]
    assert positions[:3].tolist() == [2**31 - 1 + i for i in range(3)] and positions[30003:30005].tolist() == [-4, -3]
    pos = torch.arange(5, 30005, device="cuda")
    assert torch.equal(positions[3:30003], pos + 7)
    own = table[1].long()[pos // 16]
    known = pos >= 16  # the first page was held before, and the table had none
    assert torch.equal(slots[3:30003][known], (own * 16 + pos % 16)[known])
    assert slots[30005:].tolist() == [-1] * 5


@gpu
@pytest.mark.parametrize("vocab", [60, 400, 3001, 40000])
@pytest.mark.parametrize("how", [dict(), dict(top_k=9), dict(top_p=0.9), dict(min_p=0.2)])
@pytest.mark.parametrize("temperature", [5e-324, 1e-310, 1e-40])
def test_least_temperatures_draw_the_largest(vocab, how, temperature):
    x = torch.randn((3, vocab), generator=torch.Generator().manual_seed(vocab)).cuda()
    assert (x.topk(2).values[:, 0] > x.topk(2).values[:, 1]).all()
    tokens, logprobs = ct.sample_tokens(x, torch.tensor([0.0, 0.5, 0.999], device="cuda"), temperature, **how)
    assert torch.equal(tokens, x.argmax(1)) and (logprobs == 0).all()


@gpu
def test_lists_that_overflow_in_every_row():
    """Rows whose list of candidates is too long, so that each takes a place among those put off while its waves read the
    list's length: 300 at once, the same tokens in every call."""
    g = torch.Generator().manual_seed(11)
    x = torch.randint(-4, 4, (300, 20000), generator=g).to(torch.bfloat16).cuda()  # 2500 equal ones at the top
    u = torch.rand(300, generator=g).cuda()
    first = check(x, u, p=0.95)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, ct.sample_tokens(x, u, top_p=0.95)))
    # Beside rows that draw from their list at once.
    k = torch.tensor([5, 0, 3000], dtype=torch.int32, device="cuda").repeat(100)
    check(x, u, k=k)


@gpu
def test_equal_rows_draw_the_same_token():
    """1500 equal rows, all put off, more than are worked on at a time: nuclei whose border is sought to the last bit of top_p
    draw the same token everywhere."""
    g = torch.Generator().manual_seed(5)
    last = float(np.nextafter(np.float32(1), np.float32(0)))  # draws the last id if the nucleus has it
    u = torch.full((1500,), last, device="cuda")
    for _ in range(12):
        x = 0.05 * torch.randn(40000, generator=g)
        r = int(torch.randint(600, 2500, (1,), generator=g))
        top = x.sort(descending=True).values
        x[-1] = (top[r] + top[r + 1]) / 2
        w = np.exp((x.double() - x.max().double()).numpy())
        share = math.fsum(w[x.numpy() > x[-1].item()]) / math.fsum(w)
        rows = x.expand(1500, 40000).contiguous().cuda()
        lo, hi = share - 1e-10, share + 1e-10
        while np.nextafter(lo, 1) < hi:
            mid = (lo + hi) / 2
            tokens = ct.sample_tokens(rows, u, 1.0, 0, mid)[0]
            assert (tokens == tokens[0]).all()
            lo, hi = (lo, mid) if tokens[0] == 39999 else (mid, hi)


@gpu
@pytest.mark.parametrize("vocab", [60, 5003, 50257])
def test_one_row_of_logits_for_many_draws(vocab):
    """As a prompt's for its first tokens: expanded, not copied."""
    x, _ = logits_of(1, vocab, torch.bfloat16, vocab)
    u = torch.rand(70, generator=torch.Generator().manual_seed(1)).cuda()
    for how in (dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.99, temperature=3.0), dict(top_k=torch.arange(70).int().cuda())):
        got = ct.sample_tokens(x.expand(70, vocab), u, **how)
        assert all(torch.equal(a, b) for a, b in zip(got, ct.sample_tokens(x.expand(70, vocab).contiguous(), u, **how)))
