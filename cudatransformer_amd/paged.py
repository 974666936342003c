"""Generating with a paged key / value cache over torch device tensors (ctattn_page_*, ctattn_cache_write and
ctattn_shared_prefix_fwd of include/ctattn.h).

A cache is a tensor [pages, page_size, heads, d] (any strides with contiguous heads).  ``page_reserve`` gives a
step's requests the pages that their new tokens need and says where each token goes, ``cache_write`` puts keys and
values there, ``flash_attn_shared_prefix`` attends to the prompt that a group of requests shares and to each request's own
tokens, ``page_release`` gives the pages of finished requests back.  Lengths, tables and counters stay on the device, so
that a captured step replays on what they hold.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from ._capi import _DTYPE_CODE, _check, _ptr, _stat_dtype, _stream_handle, last_error, load, on_device

_Strides10, _Strides12 = ctypes.c_int64 * 10, ctypes.c_int64 * 12


def _check_ints(name, what, t, shape, dtype, device):
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous {dtype} {list(shape)} on {device}, got {t.dtype} {list(t.shape)} "
                         f"on {t.device}")


def _check_table(name, what, t, rows, device):
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[0] != rows or t.device != device or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name}: {what} must be int32 [{rows}, pages] with contiguous rows on {device}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")


def _check_pool(name, lens, table, free, counters, page_size):
    if not lens.is_cuda or lens.dim() != 1:
        raise ValueError(f"{name}: lens must be int32 [requests] on the GPU")
    device, n = lens.device, lens.shape[0]
    _check_ints(name, "lens", lens, (n,), torch.int32, device)
    _check_table(name, "table", table, n, device)
    if free.dim() != 1:
        raise ValueError(f"{name}: free must be int32 [places]")
    _check_ints(name, "free", free, free.shape, torch.int32, device)
    _check_ints(name, "counters", counters, (2,), torch.int64, device)
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError(f"{name}: page size {page_size}, a power of two is wanted")
    return device, n


def _on(device, stream, fn, *args):
    """fn(*args) where the tensors' device is current, and `stream` if given."""
    if stream is None and device.index == torch.cuda.current_device():
        return fn(*args)
    with on_device(device, stream):
        return fn(*args)


def _given(name, what, t, make, shape, dtype, device):
    if t is None:
        return make(shape, dtype=dtype)
    _check_ints(name, what, t, shape, dtype, device)
    return t


def page_reserve(lens, new_lens, table, free, counters, page_size: int, max_tokens: int, offsets=None, out=None, stream=None):
    """(slots, positions, starts, lens, counters) of a step that adds new_lens [requests] tokens to requests of lens [requests]
    own tokens; the fresh pages are written into `table` [requests, pages], in place.

    `free` [places] is the ring of free pages and counters [2] says how many were taken from it and given to it
    (``page_pool`` makes them).  slots and positions [max_tokens] (int64) are the cache place and the number of
    each new token, offsets [requests] added; rows behind the last hold -1 and 0.  starts [requests + 1] are the requests'
    first rows.  Requests are served in order, whole or not at all: one without room keeps its length and its rows hold -1
    and 0.  `out` is a tuple of five tensors to write instead of new ones, apart from the inputs."""
    name = "page_reserve"
    device, n = _check_pool(name, lens, table, free, counters, page_size)
    _check_ints(name, "new_lens", new_lens, (n,), torch.int32, device)
    if offsets is not None:
        _check_ints(name, "offsets", offsets, (n,), torch.int32, device)
    if max_tokens < 0:
        raise ValueError(f"{name}: max_tokens {max_tokens}")
    if out is not None and len(out) != 5:
        raise ValueError(f"{name}: out must be (slots, positions, starts, lens, counters)")
    return _on(device, stream, _reserve, name, lens, new_lens, table, free, counters, page_size, max_tokens, offsets, out, device, n, stream)


def _reserve(name, lens, new_lens, table, free, counters, page_size, max_tokens, offsets, out, device, n, stream):
    want = (((max_tokens,), torch.int64), ((max_tokens,), torch.int64), ((n + 1,), torch.int32), ((n,), torch.int32), ((2,), torch.int64))
    if out is None:
        out = tuple(lens.new_empty(shape, dtype=dtype) for shape, dtype in want)
    else:
        names = "slots", "positions", "starts", "lens", "counters"
        out = tuple(_given(name, f"out's {what}", t, lens.new_empty, *w, device) for what, t, w in zip(names, out, want))
    slots, positions, starts, lens_out, counters_out = out
    rc = load().ctattn_page_reserve(lens.data_ptr(), new_lens.data_ptr(), _ptr(offsets), table.data_ptr(), free.data_ptr(),
                                    counters.data_ptr(), slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
                                    lens_out.data_ptr(), counters_out.data_ptr(), n, table.stride(0), table.shape[1], free.shape[0],
                                    page_size, max_tokens, _stream_handle(stream))
    if rc != 0:
        _check(rc, "ctattn_page_reserve")
    return out


def page_release(done, lens, table, free, counters, page_size: int, out=None, stream=None):
    """(lens, counters) after the pages of the requests with done [requests] (bool) have gone back into the ring `free`,
    in place; `out` is a tuple of two tensors to write instead of new ones, apart from the inputs."""
    name = "page_release"
    device, n = _check_pool(name, lens, table, free, counters, page_size)
    _check_ints(name, "done", done, (n,), torch.bool, device)
    if out is not None and len(out) != 2:
        raise ValueError(f"{name}: out must be (lens, counters)")
    return _on(device, stream, _release, name, done, lens, table, free, counters, page_size, out, device, n, stream)


def _release(name, done, lens, table, free, counters, page_size, out, device, n, stream):
    lens_out, counters_out = out or (None, None)
    lens_out = _given(name, "out's lens", lens_out, lens.new_empty, (n,), torch.int32, device)
    counters_out = _given(name, "out's counters", counters_out, lens.new_empty, (2,), torch.int64, device)
    rc = load().ctattn_page_release(done.data_ptr(), lens.data_ptr(), table.data_ptr(), free.data_ptr(), counters.data_ptr(),
                                    lens_out.data_ptr(), counters_out.data_ptr(), n, table.stride(0), table.shape[1],
                                    free.shape[0], page_size, _stream_handle(stream))
    if rc != 0:
        _check(rc, "ctattn_page_release")
    return lens_out, counters_out


def page_pool(pages, device="cuda"):
    """(free, counters) of a ring that holds these pages (a number of them, or a 1-D int32 tensor) as free."""
    free = torch.arange(pages, dtype=torch.int32, device=device) if isinstance(pages, int) else pages.to(device, torch.int32).clone()
    if free.dim() != 1:
        raise ValueError("page_pool: pages must be a number or a 1-D tensor")
    return free, torch.tensor([0, free.shape[0]], device=free.device)


def _check_caches(name, k_cache, v_cache, dtype, device):
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"{name}: caches must be [pages, page_size, heads, d], got {list(k_cache.shape)} and {list(v_cache.shape)}")
    for t in (k_cache, v_cache):
        if t.dtype != dtype or t.device != device:
            raise ValueError(f"{name}: caches must be {dtype} on {device}, got {t.dtype} on {t.device}")
        if t.stride(3) != 1 and t.shape[3] > 1:
            raise ValueError(f"{name}: a head's elements must be contiguous")
    page_size = k_cache.shape[1]
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError(f"{name}: page size {page_size}, a power of two is wanted")


def cache_write(k, v, k_cache, v_cache, slots, stream=None):
    """Copies k and v [rows, heads, d] (any row and head strides) to the places `slots` [rows] (int64) of the caches
    [pages, page_size, heads, d], in place; rows with a slot outside, as -1, are skipped.  Autograd does not see it: no gradient
    comes back to k and v, and the caches' versions stay."""
    name = "cache_write"
    if k.dim() != 3 or v.shape != k.shape or not k.is_cuda:
        raise ValueError(f"{name}: k and v must be [rows, heads, d] on the GPU, got {list(k.shape)} and {list(v.shape)}")
    if k.dtype not in _DTYPE_CODE or v.dtype != k.dtype or v.device != k.device:
        raise ValueError(f"{name}: k and v must be of one floating dtype on one device, got {k.dtype} and {v.dtype}")
    _check_caches(name, k_cache, v_cache, k.dtype, k.device)
    rows, heads, d = k.shape
    if tuple(k_cache.shape[2:]) != (heads, d):
        raise ValueError(f"{name}: k {list(k.shape)} does not match the caches {list(k_cache.shape)}")
    for t in (k, v):
        if t.stride(2) != 1 and d > 1:
            raise ValueError(f"{name}: a head's elements must be contiguous")
    _check_ints(name, "slots", slots, (rows,), torch.int64, k.device)
    _on(k.device, stream, _write, k, v, k_cache, v_cache, slots, rows, heads, d, stream)


def _write(k, v, k_cache, v_cache, slots, rows, heads, d, stream):
    strides = _Strides10(*k.stride()[:2], *v.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3])
    rc = load().ctattn_cache_write(_DTYPE_CODE[k.dtype], k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                   slots.data_ptr(), strides, rows, heads, d, k_cache.shape[0], k_cache.shape[1],
                                   _stream_handle(stream))
    if rc != 0:
        _check(rc, "ctattn_cache_write")


@functools.lru_cache(maxsize=256)
def _shared_prefix_need(code, *sizes):
    n = load().ctattn_shared_prefix_workspace_bytes(code, *sizes)
    if n < 0:
        raise ValueError(last_error())
    return n


def shared_prefix_workspace_bytes(dtype, rows: int, requests: int, groups: int, num_heads: int, num_kv_heads: int, d: int,
                                  page_size: int, table_width: int, prefix_width: int) -> int:
    """Bytes of the workspace of flash_attn_shared_prefix, with or without starts and group_starts."""
    return _shared_prefix_need(_DTYPE_CODE[dtype], rows, requests, groups, num_heads, num_kv_heads, d, page_size, table_width,
                               prefix_width)


def flash_attn_shared_prefix(q, k_cache, v_cache, table, lens, prefix_table=None, prefix_lens=None, group_starts=None, starts=None,
                             out=None, lse=None, workspace=None, stream=None):
    """O [rows, Hq, d] and LSE [rows, Hq] of the requests' new tokens q [rows, Hq, d] over the prompt that a group of requests
    shares and each request's own tokens; the caches are [pages, page_size, Hkv, d], Hq a multiple of Hkv.

    table [requests, pages] and lens [requests] are the requests' pages and own tokens, the new ones among them;
    prefix_table [groups, pages] and prefix_lens [groups] the prompts' (None: no prompts); int32.  group_starts [groups + 1] are
    the first requests of the groups (None: equal groups), starts [requests + 1] the first rows of the requests, whose last
    tokens the rows are (None: one row a request).  Rows of no request are left as they are in a given output, zeros (LSE -inf) in
    one allocated here.  For inference: no gradient is recorded."""
    name = "flash_attn_shared_prefix"
    if q.dim() != 3 or not q.is_cuda:
        raise ValueError(f"{name}: q must be [rows, heads, d] on the GPU, got {list(q.shape)}")
    dtype, device = q.dtype, q.device
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"{name}: dtype {dtype} unsupported (float32, bfloat16, float16, float64)")
    rows, hq, d = q.shape
    _check_caches(name, k_cache, v_cache, dtype, device)
    pages, page_size, hkv, kd = k_cache.shape
    if kd != d or hkv < 1 or hq % hkv != 0:
        raise ValueError(f"{name}: q {list(q.shape)} on caches {list(k_cache.shape)}")
    if lens.dim() != 1:
        raise ValueError(f"{name}: lens must be int32 [requests]")
    n = lens.shape[0]
    _check_ints(name, "lens", lens, (n,), torch.int32, device)
    _check_table(name, "table", table, n, device)
    if (prefix_table is None) != (prefix_lens is None):
        raise ValueError(f"{name}: prefix_table and prefix_lens go together")
    groups = 0
    if prefix_table is not None:
        groups = prefix_lens.shape[0] if prefix_lens.dim() == 1 else -1
        _check_ints(name, "prefix_lens", prefix_lens, (max(groups, 0),), torch.int32, device)
        _check_table(name, "prefix_table", prefix_table, groups, device)
        if group_starts is None and groups > 0 and n % groups != 0:
            raise ValueError(f"{name}: {n} requests in {groups} equal groups; other ones need group_starts")
    if group_starts is not None:
        _check_ints(name, "group_starts", group_starts, (groups + 1,), torch.int32, device)
    if starts is not None:
        _check_ints(name, "starts", starts, (n + 1,), torch.int32, device)
    elif rows != n:
        raise ValueError(f"{name}: {rows} rows of {n} requests; other than one a request needs starts")
    for t in (q,) if out is None else (q, out):
        if t.shape != q.shape or t.dtype != dtype or t.device != device or (t.stride(2) != 1 and d > 1):
            raise ValueError(f"{name}: q and out must be {dtype} {list(q.shape)} on {device} with contiguous heads")
    if lse is not None:
        _check_ints(name, "lse", lse, (rows, hq), _stat_dtype(dtype), device)
    if workspace is not None and (not workspace.is_contiguous() or workspace.device != device):
        raise ValueError(f"{name}: workspace must be contiguous on {device}")
    return _on(device, stream, _shared_prefix, q, k_cache, v_cache, table, lens, prefix_table, prefix_lens, group_starts, starts,
               out, lse, workspace, rows, n, groups, hq, hkv, d, pages, page_size, stream)


def _shared_prefix(q, k_cache, v_cache, table, lens, prefix_table, prefix_lens, group_starts, starts, out, lse, workspace, rows, n,
                   groups, hq, hkv, d, pages, page_size, stream):
    width, pwidth = table.shape[1], prefix_table.shape[1] if groups else 0
    # The call fills rows of no request, which only starts can leave, in both outputs or in neither.
    code, fill = _DTYPE_CODE[q.dtype], out is None and lse is None
    mixed = starts is not None and not fill
    need = _shared_prefix_need(code, rows, n, groups, hq, hkv, d, page_size, width, pwidth)
    if out is None:
        out = q.new_zeros((rows, hq, d)) if mixed else q.new_empty((rows, hq, d))
    if lse is None:
        stat = _stat_dtype(q.dtype)
        lse = q.new_full((rows, hq), -math.inf, dtype=stat) if mixed else q.new_empty((rows, hq), dtype=stat)
    if workspace is None:
        workspace = q.new_empty(max(need, 1), dtype=torch.uint8)
    strides = _Strides12(*q.stride()[:2], *out.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3], table.stride(0),
                         prefix_table.stride(0) if groups else 0)
    rc = load().ctattn_shared_prefix_fwd(code, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), lens.data_ptr(),
                                         _ptr(prefix_table), _ptr(prefix_lens), _ptr(group_starts), _ptr(starts), out.data_ptr(),
                                         lse.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(), strides,
                                         rows, n, groups, hq, hkv, d, pages, page_size, width, pwidth, int(fill),
                                         _stream_handle(stream))
    if rc != 0:
        _check(rc, "ctattn_shared_prefix_fwd")
    return out, lse


__all__ = ["cache_write", "flash_attn_shared_prefix", "page_pool", "page_release", "page_reserve",
           "shared_prefix_workspace_bytes"]
