"""What the packed entries refuse of memory that is used twice (CPU: every refusal is made before a launch)."""
import ctypes

import pytest

import cudatransformer_amd as ct
from cudatransformer_amd import _capi

BIG = 1 << 20  # places far apart
LENS, HQ, HKV, D = [5, 3], 4, 2, 64
ROWS = sum(LENS)
ESIZE = {0: 4, 1: 2, 2: 2, 3: 8}


def _plan():
    return ct.packed_plan(LENS, HQ, HKV, device="cpu")


def _strides(heads):
    return (ctypes.c_int64 * (2 * len(heads)))(*(x for h in heads for x in (h * D, D)))


def _fwd(plan, at, dtype):
    """at: q, k, v, o, lse."""
    q, k, v, o, lse = at
    rc = _capi.load().ctattn_packed_fwd(dtype, q, k, v, o, lse, _strides([HQ, HKV, HKV, HQ]), plan._host.data_ptr(), 64, ROWS, HQ,
                                        HKV, D, 1, None)
    return rc, _capi.last_error()


def _bwd(plan, at, dtype, ws=32 * BIG):
    """at: q, k, v, o, dout, lse, dq, dk, dv."""
    lib = _capi.load()
    need = lib.ctattn_packed_bwd_workspace_bytes(dtype, plan._host.data_ptr(), HQ, HKV, D)
    rc = lib.ctattn_packed_bwd(dtype, *at, ws, need, _strides([HQ, HKV, HKV, HQ, HQ, HQ, HKV, HKV]), plan._host.data_ptr(), 64, ROWS,
                               HQ, HKV, D, 1, None)
    return rc, _capi.last_error(), need


@pytest.mark.parametrize("dtype", [0, 1, 2, 3])
def test_lse_lies_on_no_tensor_of_the_forward(dtype):
    plan = _plan()
    stat = 8 if dtype == 3 else 4
    for i, heads in enumerate((HQ, HKV, HKV, HQ)):
        last = ROWS * heads * D * ESIZE[dtype] - 8  # the tensor's last 8 bytes
        for lse in ((i + 1) * BIG, (i + 1) * BIG + last, (i + 1) * BIG - ROWS * HQ * stat + 8):
            rc, said = _fwd(plan, (BIG, 2 * BIG, 3 * BIG, 4 * BIG, lse), dtype)
            assert rc == 1 and "lse lies on" in said, (i, lse)


@pytest.mark.parametrize("dtype", [0, 1, 2, 3])
def test_gradients_lie_on_no_lse_and_the_workspace_on_nothing(dtype):
    plan = _plan()
    apart = [(i + 1) * BIG for i in range(9)]
    for g in (6, 7, 8):
        at = list(apart)
        at[5] = at[g] + 64
        rc, said, need = _bwd(plan, at, dtype)
        assert rc == 1 and "input's memory" in said, g
    for i, heads in enumerate((HQ, HKV, HKV, HQ, HQ, 0, HQ, HKV, HKV)):
        size = ROWS * heads * D * ESIZE[dtype] if heads else ROWS * HQ * (8 if dtype == 3 else 4)
        for ws in (apart[i], apart[i] + (size - 1) // 16 * 16, apart[i] + 16 - (need + 15) // 16 * 16):
            rc, said, _ = _bwd(plan, apart, dtype, ws=ws)
            assert rc == 1 and "workspace lies on" in said, (i, ws)


def test_slices_of_one_buffer():
    """q and o as slices of one row-major buffer are refused where they are shifted onto each other within the rows."""
    lib, plan = _capi.load(), _plan()
    host, es, row = plan._host.data_ptr(), 2, 2 * HQ * D

    def call(o_at):
        st = (ctypes.c_int64 * 8)(row, D, HKV * D, D, HKV * D, D, row, D)
        rc = lib.ctattn_packed_fwd(1, BIG, 4 * BIG, 5 * BIG, BIG + es * o_at, None, st, host, 64, ROWS, HQ, HKV, D, 1, None)
        return rc, _capi.last_error()

    # One element into q's part of a row, at either end, and half of the part.
    for o_at in (0, 1, HQ * D - 1, HQ * D // 2, HQ * D + 1, row - 1, -1, 1 - HQ * D):
        rc, said = call(o_at)
        assert rc == 1 and "input's memory" in said, o_at
