"""Scaled token lookup and its gradient by sorted tokens over torch device tensors
(ctattn_embedding_lookup / ctattn_embedding_grad of include/ctattn.h)."""
from __future__ import annotations

import torch

from ._capi import _DTYPE_CODE, _check, _ptr, _stream_handle, last_error, load, on_device

_ID_CODE = {torch.int32: 4, torch.int64: 5}  # CTATTN_I32, CTATTN_I64


def _check_rows(name, ids, *ts):
    if ids.dtype not in _ID_CODE or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError(f"{name}: ids must be contiguous int32 or int64 on the GPU")
    for t in ts:
        if t.dtype not in _DTYPE_CODE or t.dtype != ts[0].dtype or t.device != ids.device or not t.is_contiguous():
            raise ValueError(f"{name}: tensors must be contiguous, of one floating dtype, on {ids.device}")


def embedding_lookup(ids, table, scale: float = 1.0, out=None, stream=None):
    """scale * table[ids], [*ids.shape, D]; an id outside the table gives zeros."""
    name = "embedding_lookup"
    _check_rows(name, ids, table, *(() if out is None else (out,)))
    if table.dim() != 2 or 0 in table.shape:
        raise ValueError(f"{name}: table must be [vocab, D], got {tuple(table.shape)}")
    vocab, d = table.shape
    shape = (*ids.shape, d)
    if out is not None and tuple(out.shape) != shape:
        raise ValueError(f"{name}: out must be {list(shape)}, got {tuple(out.shape)}")
    with on_device(ids.device, stream):
        out = table.new_empty(shape) if out is None else out
        rc = load().ctattn_embedding_lookup(_DTYPE_CODE[table.dtype], _ID_CODE[ids.dtype], _ptr(ids), _ptr(table),
                                            _ptr(out), float(scale), ids.numel(), d, vocab, _stream_handle(stream))
    _check(rc, "ctattn_embedding_lookup")
    return out


def embedding_grad_workspace_bytes(dtype, n: int, d: int, vocab: int) -> int:
    """Bytes of the workspace of embedding_grad for n ids."""
    need = load().ctattn_embedding_grad_workspace_bytes(_DTYPE_CODE[dtype], n, d, vocab)
    if need < 0:
        raise ValueError(last_error())
    return need


def embedding_grad(ids, dout, vocab: int, scale: float = 1.0, out=None, accumulate: bool = False, workspace=None,
                   stream=None):
    """The gradient [vocab, D] of embedding_lookup's table from dout [*ids.shape, D]: every row, in the
    order of the tokens' positions; with accumulate added to what `out` holds."""
    name = "embedding_grad"
    _check_rows(name, ids, dout, *(() if out is None else (out,)))
    if dout.dim() != ids.dim() + 1 or dout.shape[:-1] != ids.shape or dout.shape[-1] < 1:
        raise ValueError(f"{name}: dout {tuple(dout.shape)} does not match ids {tuple(ids.shape)}")
    d = dout.shape[-1]
    if accumulate and out is None:
        raise ValueError(f"{name}: accumulate needs the gradient to add to")
    if out is not None and tuple(out.shape) != (vocab, d):
        raise ValueError(f"{name}: out must be {[vocab, d]}, got {tuple(out.shape)}")
    need = embedding_grad_workspace_bytes(dout.dtype, ids.numel(), d, vocab)
    with on_device(ids.device, stream):
        out = dout.new_empty((vocab, d)) if out is None else out
        if workspace is None:
            workspace = dout.new_empty(max(need, 1), dtype=torch.uint8)
        elif not workspace.is_contiguous() or workspace.device != ids.device:
            raise ValueError(f"{name}: workspace must be contiguous on {ids.device}")
        rc = load().ctattn_embedding_grad(_DTYPE_CODE[dout.dtype], _ID_CODE[ids.dtype], _ptr(ids), _ptr(dout), _ptr(out),
                                          float(scale), int(bool(accumulate)), _ptr(workspace),
                                          workspace.numel() * workspace.element_size(), ids.numel(), d, vocab,
                                          _stream_handle(stream))
    _check(rc, "ctattn_embedding_grad")
    return out


class EmbeddingLookupFunction(torch.autograd.Function):
    """torch.autograd wrapper: forward and backward both run the ctattn kernels."""

    @staticmethod
    def forward(ctx, ids, table, scale=1.0):
        ids = ids.contiguous()
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = table.shape[0], scale
        return embedding_lookup(ids, table.contiguous(), scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        return None, embedding_grad(ids, dout.contiguous(), ctx.vocab, ctx.scale), None


def embedding(ids, table, scale: float = 1.0):
    """Differentiable scale * table[ids] on the ctattn kernels."""
    return EmbeddingLookupFunction.apply(ids, table, scale)


__all__ = ["EmbeddingLookupFunction", "embedding", "embedding_grad", "embedding_grad_workspace_bytes",
           "embedding_lookup"]
