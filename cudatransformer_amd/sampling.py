"""Next tokens from logits and given random numbers over torch device tensors (ctattn_sample of include/ctattn.h)."""
from __future__ import annotations

import functools
import operator

import torch

from ._capi import _DTYPE_CODE, _check, _ptr, _stream_handle, last_error, load, on_device


@functools.lru_cache(maxsize=256)
def _need(rows, vocab):
    need = load().ctattn_sample_workspace_bytes(rows, vocab)
    if need < 0:
        raise ValueError(last_error())
    return need


def sample_workspace_bytes(rows: int, vocab: int) -> int:
    """Bytes of the workspace of sample_tokens."""
    return _need(rows, vocab)


def sample_tokens(logits, u=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, tokens=None, logprobs=None, workspace=None,
                  stream=None):
    """(tokens, logprobs) [rows]: a token (int64) of each row of logits [rows, vocab] (float32, bfloat16 or float16; rows
    apart or one expanded) from random numbers u [rows] (float32 in [0, 1)), and its log-probability (float32) among all tokens at
    the row's temperature.

    Tokens are ranked by logit, equal ones by the lower id.  Kept are the first top_k (0: all), of these the ranks
    before which less than top_p of their probability lies (1: all), of these the ones at least min_p times as
    probable as the first; always the first.  A token is drawn in the order of ids.  temperature <= 0 takes the first
    rank.  Each parameter is a number or a tensor [rows] (float32; top_k int32).  Logits of -inf or NaN are
    never taken; a row of nothing else gives token -1."""
    name = "sample_tokens"
    if logits.dim() != 2 or not logits.is_cuda or logits.shape[1] < 1 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"{name}: logits must be [rows, vocab] with contiguous rows on the GPU, got {list(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"{name}: dtype {logits.dtype} unsupported (float32, bfloat16, float16)")
    (rows, vocab), device = logits.shape, logits.device

    def check(what, x, dtype):
        if x.dtype is not dtype or x.shape != (rows,) or x.device != device or not x.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous {dtype} [{rows}] on {device}, got {x.dtype} {list(x.shape)} on "
                             f"{x.device}")

    def each(what, x, dtype, number):
        if not isinstance(x, torch.Tensor):
            return None, number(x)
        check(what, x, dtype)
        return x, number(0)

    t, t_all = each("temperature", temperature, torch.float32, float)
    k, k_all = each("top_k", top_k, torch.int32, operator.index)
    p, p_all = each("top_p", top_p, torch.float32, float)
    m, m_all = each("min_p", min_p, torch.float32, float)
    if u is None:
        if t is not None or t_all > 0:
            raise ValueError(f"{name}: random numbers may be left out for temperature 0 alone")
    else:
        if not isinstance(u, torch.Tensor):
            raise ValueError(f"{name}: u must be a tensor")
        check("u", u, torch.float32)
    if tokens is not None:
        check("tokens", tokens, torch.int64)
    if logprobs is not None:
        check("logprobs", logprobs, torch.float32)
    if workspace is not None and (not workspace.is_contiguous() or workspace.device != device):
        raise ValueError(f"{name}: workspace must be contiguous on {device}")
    if stream is None and device.index == torch.cuda.current_device():
        return _sample(logits, u, t, k, p, m, t_all, k_all, p_all, m_all, tokens, logprobs, workspace, rows, vocab, None)
    with on_device(device, stream):
        return _sample(logits, u, t, k, p, m, t_all, k_all, p_all, m_all, tokens, logprobs, workspace, rows, vocab, stream)


def _sample(logits, u, t, k, p, m, t_all, k_all, p_all, m_all, tokens, logprobs, workspace, rows, vocab, stream):
    need = _need(rows, vocab)
    tokens = logits.new_empty(rows, dtype=torch.int64) if tokens is None else tokens
    logprobs = logits.new_empty(rows, dtype=torch.float32) if logprobs is None else logprobs
    if workspace is None and need > 0:
        workspace = logits.new_empty(need, dtype=torch.uint8)
    rc = load().ctattn_sample(_DTYPE_CODE[logits.dtype], logits.data_ptr(), _ptr(u), _ptr(t), _ptr(k), _ptr(p), _ptr(m), t_all, k_all,
                              p_all, m_all, tokens.data_ptr(), logprobs.data_ptr(), _ptr(workspace),
                              0 if workspace is None else workspace.numel() * workspace.element_size(), rows, vocab,
                              logits.stride(0), _stream_handle(stream))
    if rc != 0:
        _check(rc, "ctattn_sample")
    return tokens, logprobs


__all__ = ["sample_tokens", "sample_workspace_bytes"]
