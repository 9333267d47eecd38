"""Dropout whose mask is never stored.

Element ``i`` (row-major over the tensor's shape) stays or goes by a pure function of
``(seed, substream, first_index + i)``: the counter generator of ``flextrain_amd.synth``, 48 bits per
element, the same for every type, layout and split of a tensor. The backward pass makes the mask again
instead of reading it. Give every call of a step its own ``substream`` (or range of indices) and every
step its own ``seed``.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _C
from .rows import Seed, dropout_record, enqueue, gpu_index, refuse_leaves, row_stride, with_even_rows, written


def dropout(x: Tensor, p: float, seed: Seed, *, substream: int = 0, first_index: int = 0, residual: Optional[Tensor] = None,
            out: Optional[Tensor] = None) -> Tensor:
    """``[residual +] keep * x / (1 - p)``, differentiable in ``x`` and ``residual``, any number of times.

    ``x``: fp32 / fp16 / bf16 GPU tensor whose rows (last dimension) lie at one distance. ``residual``
    has x's shape; its type is the result's (without one, x's is). ``seed``: a number, or one int64
    element of GPU memory -- then a pass recorded into a HIP graph follows a seed that changes between
    replays; it must keep its value until the backward pass has run. ``out`` (no gradients then) may be
    ``x`` or ``residual``, or memory of its own. A dropped element contributes 0 even where ``x`` is inf or nan.
    """
    if out is None and torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, float(p), seed, substream, first_index, seed if isinstance(seed, Tensor) else None, None)
    if out is not None:
        refuse_leaves("out", x, residual, out)
    return _apply(x, float(p), seed, substream, first_index, residual, out)


def _apply(x: Tensor, p: float, seed: Seed, substream: int, first_index: int, residual: Optional[Tensor] = None, out: Optional[Tensor] = None,
           dtype: Optional[torch.dtype] = None) -> Tensor:
    index = gpu_index(x=x, residual=residual, out=out)
    shape = x.shape
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual has shape {tuple(residual.shape)}, x {tuple(shape)}")
    if dtype is None:
        dtype = x.dtype if residual is None else residual.dtype
    cols = shape[-1] if shape else 1
    given = out
    if out is None:
        out, out_stride = x.new_empty(shape, dtype=dtype), cols
    elif out.shape != shape or out.dtype != dtype:
        raise ValueError(f"out must have shape {tuple(shape)} and type {dtype}")
    else:
        out_stride = row_stride("out", out, cols)
    rows = x.numel() // cols if cols else 0
    enqueue("ft_dropout", _C.lib().ft_dropout, index,
            x.data_ptr(), _C.dtype_code(x.dtype), row_stride("x", x, cols),
            None if residual is None else residual.data_ptr(), 0 if residual is None else row_stride("residual", residual, cols),
            out.data_ptr(), _C.dtype_code(dtype), out_stride, rows, cols,
            ctypes.byref(dropout_record(index, p, seed, substream, first_index)))
    return out if given is None else written(out)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, substream, first_index, seed_tensor, dtype):
        ctx.save_for_backward(seed_tensor)  # a seed that changes before the backward pass is found out
        ctx.mask = (p, seed, substream, first_index)
        ctx.x_dtype = x.dtype
        return _apply(x, p, seed, substream, first_index, residual, dtype=dtype)

    @staticmethod
    def backward(ctx, dy):
        (seed_tensor,) = ctx.saved_tensors
        p, seed, substream, first_index = ctx.mask
        dx = None
        if ctx.needs_input_grad[0]:
            g = with_even_rows(dy)
            if torch.is_grad_enabled() and g.requires_grad:  # linear: the gradient of the gradient is the operator again
                dx = _Dropout.apply(g, None, p, seed, substream, first_index, seed_tensor, ctx.x_dtype)
            else:
                dx = _apply(g, p, seed if seed_tensor is None else seed_tensor, substream, first_index, dtype=ctx.x_dtype)
        return (dx, dy if ctx.needs_input_grad[1] else None) + (None,) * 6
