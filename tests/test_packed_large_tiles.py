"""Attention on packed sequences where a batch has work enough for the larger tiles in every kernel, causal and not: the
forward's and dQ's of 128 rows, dK's and dV's of 128 keys, whose two slices of rows join at the end.  Bounds as in
test_packed_attention."""
import pytest
import torch

import cudatransformer_amd as ct
from test_packed_attention import _check, _inputs, _reference, _run

LENS = [512, 449, 500, 33, 512, 511, 480, 1] * 6
HQ, HKV = 16, 4


def _blocks_per_slot(causal, walk, slots):
    """Blocks of 128 x 64 pairs for each workgroup that the chip holds, over the longest workgroup's: the larger tiles are
    taken above 1/4 of it (dK, dV of 256-byte rows: 1/8)."""
    pairs = sum(n * (n + 1) // 2 if causal else n * n for n in LENS) * HQ
    return pairs / (128 * 64 * slots * walk)


def test_the_batch_is_past_the_rule():
    cus, group, longest = 256, HQ // HKV, max(LENS)
    for causal in (True, False):
        assert _blocks_per_slot(causal, -(-longest // 64), 2 * cus) > 1.5 / 4  # forward, dQ
        assert _blocks_per_slot(causal, -(-longest * group // 64), 2 * cus) > 1.5 / 4  # dK, dV, rows to 128 bytes
        assert _blocks_per_slot(causal, -(-longest * group // 64), cus) > 1.5 / 4  # dK, dV, longer rows


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 24), (torch.bfloat16, 56),
                                     (torch.bfloat16, 128), (torch.bfloat16, 104), (torch.float16, 32), (torch.float16, 64),
                                     (torch.float16, 40), (torch.float16, 128), (torch.float32, 32), (torch.float32, 64),
                                     (torch.float32, 28), (torch.float32, 52), (torch.float32, 128)])
def test_larger_tiles(dtype, d, causal):
    x = _inputs(LENS, HQ, HKV, d, dtype, seed=d)
    plan = ct.packed_plan(LENS, HQ, HKV)
    _check(_run(*x, plan, causal), _reference(*x, LENS, causal), dtype, plan.tokens)
