"""Embedding rows and their gradient, next to the optimizer that owns the table.

``embedding_lookup`` gathers scaled rows of a table (optionally dropped out in the same pass);
``embedding_grad_`` adds the lookup's gradient into a gradient accumulator, touching only the rows that
a token names, where torch makes a dense gradient of the whole table and the reference's hook adds that
to the accumulator (``flextrain/optimizer.py:194-215``). ``embedding`` is the two of them for autograd;
``FlexTrainOptimizer.embedding`` calls it with the optimizer's own accumulator.

Ids outside ``first_row ... first_row + rows - 1`` are those of other shards of the vocabulary: their
rows read as zero (so that the shards' results add up to the whole) and have no gradient.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _C
from .rows import Seed, dropout_record, enqueue, gpu_index, order_of, refuse_leaves, refuse_tangents, row_stride, token_record, with_even_rows, written


def _table(name: str, t: Tensor) -> int:
    """Row stride of a table or an accumulator."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, not {t.dim()}")
    return row_stride(name, t, t.shape[1])


def embedding_lookup(tokens: Tensor, table: Tensor, *, scale: float = 1.0, first_row: int = 0, dropout: float = 0.0, seed: Seed = 0,
                     substream: int = 0, first_index: int = 0, dtype: Optional[torch.dtype] = None, out: Optional[Tensor] = None) -> Tensor:
    """``dropout(scale * table[tokens - first_row])`` without gradients, in ``dtype`` (the table's by
    default), shape ``tokens.shape + (table.shape[1],)``.

    ``tokens``: int64 or int32, of any shape where contiguous, else of one or two dimensions with any
    strides (``batch[:, :-1]``). One fp32 product per element, rounded once. Dropout as in
    ``flextrain_amd.dropout_mask``: element ``i`` of the result is element ``first_index + i`` of
    ``(seed, substream)``."""
    index = gpu_index(table=table, tokens=tokens, out=out)
    table_stride = _table("table", table)
    rows, cols = table.shape
    shape = (*tokens.shape, cols)
    given = out
    if out is not None and out.requires_grad:
        refuse_leaves("out", out)
    if out is None:
        out, out_stride = table.new_empty(shape, dtype=dtype), cols
    elif out.shape != shape or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out must have shape {shape}" + ("" if dtype is None else f" and type {dtype}"))
    else:
        out_stride = row_stride("out", out, cols)
    record, _ = token_record(tokens, first_row, None)
    enqueue("ft_embedding_lookup", _C.lib().ft_embedding_lookup, index,
            ctypes.byref(record), table.data_ptr(), _C.dtype_code(table.dtype), rows, table_stride, out.data_ptr(), _C.dtype_code(out.dtype),
            out_stride, cols, scale,
            None if dropout == 0.0 else ctypes.byref(dropout_record(index, dropout, seed, substream, first_index)))
    return out if given is None else written(out)


def embedding_grad_(acc: Tensor, tokens: Tensor, grads: Tensor, *, scale: float = 1.0, first_row: int = 0, padding_token: Optional[int] = None,
                    accumulate: bool = True, dropout: float = 0.0, seed: Seed = 0, substream: int = 0, first_index: int = 0) -> Tensor:
    """``acc[v] += scale * (sum of the rows of grads whose token is v)`` in place; returns ``acc``.

    ``grads`` holds one row per token (``tokens.shape + (acc.shape[1],)``); tokens equal to
    ``padding_token`` add nothing. ``accumulate=False`` writes the gradient instead: the sums, and zeros
    in every row without a token. With ``dropout`` the mask of the lookup that had the same values is
    applied to ``grads`` first. Sums are kept in fp32 and rounded to acc's type once; the same call
    gives the same bits."""
    index = gpu_index(acc=acc, tokens=tokens, grads=grads)
    if acc.requires_grad:
        refuse_leaves("acc", acc)
    acc_stride = _table("acc", acc)
    rows, cols = acc.shape
    if grads.shape != (*tokens.shape, cols):
        raise ValueError(f"grads have shape {tuple(grads.shape)}, tokens {tuple(tokens.shape)} and acc {tuple(acc.shape)}")
    record, n = token_record(tokens, first_row, padding_token)
    lib = _C.lib()
    need = lib.ft_embedding_grad_workspace_bytes(n, rows, cols)
    workspace = torch.empty(need, dtype=torch.uint8, device=acc.device) if need else None
    enqueue("ft_embedding_grad", lib.ft_embedding_grad, index,
            ctypes.byref(record), grads.data_ptr(), _C.dtype_code(grads.dtype), row_stride("grads", grads, cols), acc.data_ptr(),
            _C.dtype_code(acc.dtype), rows, acc_stride, cols, scale, int(bool(accumulate)),
            None if dropout == 0.0 else ctypes.byref(dropout_record(index, dropout, seed, substream, first_index)),
            None if workspace is None else workspace.data_ptr(), need)
    return written(acc)


def embedding(tokens: Tensor, weight: Tensor, *, scale: float = 1.0, first_row: int = 0, padding_token: Optional[int] = None,
              dropout: float = 0.0, seed: Seed = 0, substream: int = 0, first_index: int = 0, dtype: Optional[torch.dtype] = None,
              grad_into: Optional[Tensor] = None) -> Tensor:
    """``embedding_lookup`` for autograd. ``weight`` gets a dense gradient of its own type -- or, with
    ``grad_into`` (shape of ``weight``, fp32 / fp16 / bf16), none: the backward pass then adds the
    gradient there, row by row, behind whatever else adds into that memory. Hooks of ``weight`` do not
    run in that case, and a backward pass confined to some leaves (``inputs=``) does not get there.

    A ``seed`` in GPU memory, and the tokens, must keep their values until the backward pass has run."""
    refuse_tangents(weight=weight)  # detach() below would drop it
    if grad_into is not None:
        gpu_index(weight=weight, grad_into=grad_into)
        if grad_into.shape != weight.shape:
            raise ValueError(f"grad_into has shape {tuple(grad_into.shape)}, weight {tuple(weight.shape)}")
        _table("grad_into", grad_into)
        _C.dtype_code(grad_into.dtype)
    if not torch.is_grad_enabled() or (grad_into is None and not weight.requires_grad):
        return embedding_lookup(tokens, weight.detach(), scale=scale, first_row=first_row, dropout=dropout, seed=seed, substream=substream,
                                first_index=first_index, dtype=dtype)
    anchor = None
    if grad_into is not None:
        # Nothing that requires a gradient goes into the lookup, yet its backward pass has to run. The
        # leaf that asks for it is new in every call: one that lived on would tie the graphs of
        # different calls (an eager one and one that is being recorded) to one stream. It is on the
        # table's GPU: at the end of a backward pass autograd makes the caller's stream wait for the
        # streams of the leaves, which for this one is the stream that the gradient is added on.
        weight, anchor = weight.detach(), torch.empty(0, device=weight.device, requires_grad=True)
    mask = (dropout, seed, substream, first_index)
    return _Embedding.apply(weight, anchor, tokens, seed if isinstance(seed, Tensor) else None, scale, first_row, padding_token, mask, dtype,
                            grad_into)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, anchor, tokens, seed_tensor, scale, first_row, padding_token, mask, dtype, grad_into):
        ctx.save_for_backward(tokens, seed_tensor)  # either changing before the backward pass is found out
        ctx.options = (scale, first_row, padding_token, mask)
        ctx.grad_into = grad_into
        ctx.weight = (weight.shape, weight.dtype, weight.device)
        p, seed, substream, first_index = mask
        return embedding_lookup(tokens, weight, scale=scale, first_row=first_row, dropout=p, seed=seed, substream=substream,
                                first_index=first_index, dtype=dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        tokens, seed_tensor = ctx.saved_tensors
        scale, first_row, padding_token, (p, seed, substream, first_index) = ctx.options
        shape, dtype, device = ctx.weight
        into = ctx.grad_into
        options = dict(scale=scale, first_row=first_row, padding_token=padding_token, dropout=p, seed=seed if seed_tensor is None else seed_tensor,
                       substream=substream, first_index=first_index)
        if into is None:
            grad = embedding_grad_(torch.empty(shape, dtype=dtype, device=device), tokens, with_even_rows(dy), accumulate=False, **options)
            return (grad,) + (None,) * 9
        with order_of(into):  # the lookups of one table may be on different streams
            embedding_grad_(into, tokens, with_even_rows(dy), **options)
        return (None,) * 10
