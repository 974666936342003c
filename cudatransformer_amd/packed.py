"""Attention on packed sequences over torch device tensors (ctattn_packed_* of include/ctattn.h).

Documents of different lengths lie one behind the other in [tokens, heads, d] tensors and attend
each to itself; several query heads may share a key / value head.  ``packed_plan`` makes the
batch's plan from its lengths, once for all layers and both directions.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from ._capi import _DTYPE_CODE, _check, _ptr, _stat_dtype, _stream_handle, last_error, load, on_device


class PackedPlan:
    """Where a packed batch's sequences begin and which tiles of them the kernels work on.

    Made on the current stream of `device`; a call on another stream waits for it.  A captured graph
    that uses a plan needs it alive and replays that plan's lengths."""

    def __init__(self, seqlens, num_heads: int, num_kv_heads: int, device="cuda"):
        if num_heads < 1 or num_kv_heads < 1 or num_heads % num_kv_heads != 0:
            raise ValueError(f"packed_plan: {num_heads} query heads on {num_kv_heads} key heads")
        if isinstance(seqlens, torch.Tensor):
            if seqlens.dim() != 1 or seqlens.is_floating_point() or seqlens.dtype == torch.bool:
                raise ValueError("packed_plan: seqlens must be a list or a 1-D integer tensor")
            seqlens = seqlens.tolist()
        try:
            self.seqlens = tuple(operator.index(n) for n in seqlens)
        except TypeError:
            raise ValueError("packed_plan: seqlens must be whole numbers") from None
        self.tokens = sum(self.seqlens)
        self.group = num_heads // num_kv_heads
        lib = load()
        n = len(self.seqlens)
        lens = (ctypes.c_int64 * max(n, 1))(*self.seqlens)
        need = lib.ctattn_packed_plan_bytes(lens, n, self.group)
        if need < 0:
            raise ValueError(last_error())
        self._positions = {}
        self.device = torch.device(device)
        if self.device.type != "cuda":
            # A plan for the host alone: its lengths and offsets, no device copy to run kernels with.
            self._host, self._dev = torch.zeros(need, dtype=torch.uint8), None
            _check(lib.ctattn_packed_plan(lens, n, self.group, self._host.data_ptr(), need), "ctattn_packed_plan")
            return
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("packed_plan: a plan is made before a graph's capture, not in it")
        self._host = torch.empty(need, dtype=torch.uint8, pin_memory=True)
        _check(lib.ctattn_packed_plan(lens, n, self.group, self._host.data_ptr(), need), "ctattn_packed_plan")
        with on_device(self.device):
            self._dev = self._host.to(self.device, non_blocking=True)
            self._ready = torch.cuda.current_stream().record_event()
            self._stream = _stream_handle(None)
        self._addresses = self._host.data_ptr(), self._dev.data_ptr()

    @property
    def cu_seqlens(self):
        """First token of each sequence and, at the end, the number of tokens."""
        out = [0]
        for n in self.seqlens:
            out.append(out[-1] + n)
        return out

    def positions(self, device=None):
        """int64 [tokens]: each token's position in its sequence (made on first use for a device, then kept; before a
        graph's capture, not in it)."""
        device = self.device if device is None else torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        capturing = device.type == "cuda" and torch.cuda.is_current_stream_capturing()
        if device not in self._positions:
            if capturing:
                raise RuntimeError("PackedPlan.positions: made before a graph's capture, not in it")
            p = torch.cat([torch.arange(n) for n in self.seqlens]) if self.seqlens else torch.empty(0, dtype=torch.int64)
            self._positions[device] = p.to(device)
        p = self._positions[device]
        if p.is_cuda and not capturing:  # the memory goes back when this stream, too, has passed what reads it
            p.record_stream(torch.cuda.current_stream(device))
        return p

    def _pointers(self, handle: int):
        if handle != self._stream:
            cur = torch.cuda.current_stream()
            if not torch.cuda.is_current_stream_capturing():  # a capture begins with a device-wide wait
                cur.wait_event(self._ready)
                self._dev.record_stream(cur)
        return self._addresses


def packed_plan(seqlens, num_heads: int, num_kv_heads: int | None = None, device="cuda") -> PackedPlan:
    """The plan of a batch of sequences of these lengths (a list or an integer tensor), for
    `num_heads` query heads on `num_kv_heads` key / value heads (as many if not given)."""
    return PackedPlan(seqlens, num_heads, num_heads if num_kv_heads is None else num_kv_heads, device)


def _check_packed(name, plan, q, k, v, *like_q):
    if not isinstance(plan, PackedPlan) or plan._dev is None:
        raise ValueError(f"{name}: plan must be a packed_plan on the GPU")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"{name}: tensors must be [tokens, heads, d], got {tuple(q.shape)} and {tuple(k.shape)}")
    dtype, device, shape = q.dtype, plan.device, q.shape
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"{name}: dtype {dtype} unsupported (float32, bfloat16, float16, float64)")
    rows, hq, d = shape
    krows, hkv, kd = kshape = k.shape
    if krows != rows or kd != d or v.shape != kshape:
        raise ValueError(f"{name}: q {tuple(shape)}, k {tuple(kshape)}, v {tuple(v.shape)} do not match")
    if hkv < 1 or hq != hkv * plan.group:
        raise ValueError(f"{name}: {hq} query heads on {hkv} key heads, the plan has {plan.group} to one")
    if rows < plan.tokens:
        raise ValueError(f"{name}: tensors of {rows} rows, the plan has {plan.tokens} tokens")
    for t in (q, k, v, *like_q):
        if t.device != device:
            raise ValueError(f"{name}: a tensor on {t.device}, the plan on {device}")
        if t.dtype != dtype:
            raise ValueError(f"{name}: dtypes differ, {t.dtype} and {dtype}")
        if t.stride(2) != 1 and d > 1:
            raise ValueError(f"{name}: a head's elements must be contiguous")
    for t in like_q:
        if t.shape != shape:
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def _check_lse(name, lse, q):
    want = (q.shape[0], q.shape[1])
    if lse.dtype != _stat_dtype(q.dtype) or tuple(lse.shape) != want or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError(f"{name}: lse must be contiguous {_stat_dtype(q.dtype)} {list(want)}")


_Strides4, _Strides8 = ctypes.c_int64 * 8, ctypes.c_int64 * 16  # (row, head) of 4 and of 8 tensors


def flash_attn_packed_fwd(q, k, v, plan, causal: bool = False, out=None, lse=None, stream=None):
    """O [rows, Hq, d] and LSE [rows, Hq] of attention within each of the plan's sequences; q [rows, Hq, d],
    k and v [rows, Hkv, d], of any row and head strides.  Rows behind the last sequence are left as they
    are (zeros where the output is allocated here)."""
    name = "flash_attn_packed_fwd"
    if out is None:
        _check_packed(name, plan, q, k, v)
    else:
        _check_packed(name, plan, q, k, v, out)
    if lse is not None:
        _check_lse(name, lse, q)
    if stream is None and plan.device.index == torch.cuda.current_device():
        return _fwd(q, k, v, plan, causal, out, lse, None)
    with on_device(plan.device, stream):
        return _fwd(q, k, v, plan, causal, out, lse, stream)


def _fwd(q, k, v, plan, causal, out, lse, stream):
    rows, hq, d = q.shape
    make = q.new_empty if rows == plan.tokens else q.new_zeros
    if out is None:
        out = make((rows, hq, d))
    if lse is None:
        lse = make((rows, hq), dtype=_stat_dtype(q.dtype))
    handle = _stream_handle(stream)
    host, dev = plan._pointers(handle)
    strides = _Strides4(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0),
                        out.stride(1))
    rc = load().ctattn_packed_fwd(_DTYPE_CODE[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                  lse.data_ptr(), strides, host, dev, rows, hq, k.shape[1], d, int(bool(causal)), handle)
    if rc != 0:
        _check(rc, "ctattn_packed_fwd")
    return out, lse


def packed_bwd_workspace_bytes(dtype, plan, num_heads: int, num_kv_heads: int, d: int) -> int:
    """Bytes of the workspace of flash_attn_packed_bwd."""
    n = load().ctattn_packed_bwd_workspace_bytes(_DTYPE_CODE[dtype], plan._host.data_ptr(), num_heads, num_kv_heads, d)
    if n < 0:
        raise ValueError(last_error())
    return n


def flash_attn_packed_bwd(q, k, v, o, do, lse, plan, causal: bool = False, dq=None, dk=None, dv=None, workspace=None,
                          stream=None):
    """dQ, dK, dV given the forward's O and LSE and the upstream dO; dK and dV sum over the query heads that
    share a key head.  Rows behind the last sequence are left as they are (zeros where allocated here)."""
    name = "flash_attn_packed_bwd"
    _check_packed(name, plan, q, k, v, o, do, *(() if dq is None else (dq,)))
    _check_lse(name, lse, q)
    rows, hq, d = q.shape
    hkv = k.shape[1]
    for g in (dk, dv):
        if g is not None and (g.shape != k.shape or g.dtype != q.dtype or g.device != q.device or (g.stride(2) != 1 and d > 1)):
            raise ValueError(f"{name}: dk and dv must be {q.dtype} {list(k.shape)} with contiguous heads")
    need = packed_bwd_workspace_bytes(q.dtype, plan, hq, hkv, d)
    with on_device(plan.device, stream):
        make = q.new_empty if rows == plan.tokens else q.new_zeros
        dq = make((rows, hq, d)) if dq is None else dq
        dk = make((rows, hkv, d)) if dk is None else dk
        dv = make((rows, hkv, d)) if dv is None else dv
        if workspace is None:
            workspace = q.new_empty(max(need, 1), dtype=torch.uint8)
        elif not workspace.is_contiguous() or workspace.device != q.device:
            raise ValueError(f"{name}: workspace must be contiguous on {q.device}")
        handle = _stream_handle(stream)
        host, dev = plan._pointers(handle)
        rc = load().ctattn_packed_bwd(_DTYPE_CODE[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                      do.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                      _ptr(workspace), workspace.numel() * workspace.element_size(),
                                      _Strides8(*(n for t in (q, k, v, o, do, dq, dk, dv) for n in t.stride()[:2])), host, dev, rows, hq, hkv, d,
                                      int(bool(causal)), handle)
    _check(rc, "ctattn_packed_bwd")
    return dq, dk, dv


def _ready(t):
    """`t`, or a copy of it where a head is not contiguous or rows lie off the 16 bytes of the fast kernels."""
    e = t.element_size()
    on16 = all(n <= 1 or step * e % 16 == 0 for n, step in zip(t.shape[:2], t.stride()[:2]))
    if t.stride(2) == 1 and t.data_ptr() % 16 == 0 and on16:
        return t
    return t.clone(memory_format=torch.contiguous_format)


class PackedAttentionFunction(torch.autograd.Function):
    """torch.autograd wrapper: forward and backward both run the ctattn kernels."""

    @staticmethod
    def forward(ctx, q, k, v, plan, causal=False):
        q, k, v = _ready(q), _ready(k), _ready(v)
        o, lse = flash_attn_packed_fwd(q, k, v, plan, causal)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.plan, ctx.causal = plan, causal
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        dq, dk, dv = flash_attn_packed_bwd(q, k, v, o, _ready(do), lse, ctx.plan, ctx.causal)
        return dq, dk, dv, None, None


def flash_attention_packed(q, k, v, plan, causal: bool = False):
    """Differentiable attention within each of the plan's sequences on the ctattn kernels."""
    return PackedAttentionFunction.apply(q, k, v, plan, causal)


__all__ = ["PackedAttentionFunction", "PackedPlan", "flash_attention_packed", "flash_attn_packed_bwd",
           "flash_attn_packed_fwd", "packed_bwd_workspace_bytes", "packed_plan"]
