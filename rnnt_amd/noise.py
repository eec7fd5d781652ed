"""Dropout with a counter-based mask that is never stored (the Dropout layers of reference rnnt/keras_model.py:102-103).

The mask is a function of (seed, offset, row, column) alone: the backward pass draws it again, and so can any other code
(``dense`` draws the same one in its epilogue).  Element (r, c) of x seen as [rows, last dimension] takes 16 bits of
Philox4x32-10 at counter (c // 8, r, offset) under the key seed; it is kept when they are >= round(rate * 65536) and then
multiplied by 65536 / (65536 - round(rate * 65536)).  A dropped infinity or NaN becomes 0.
"""
from __future__ import annotations

import torch

from . import _lib
from ._operator import check, drop16, dtype_code, need_gpu, on_device, seed_offset, stream


def _rows(x):
    """x as rows of its last dimension: (tensor to read, rows, columns, row stride).  One-dimensional rows may be any
    distance apart; anything else is made dense."""
    cols = x.shape[-1]
    if x.dim() == 1:
        return (x if x.stride(0) == 1 else x.contiguous()), 1, cols, cols
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= cols:
        return x, x.shape[0], cols, x.stride(0)
    x = x.contiguous()
    return x, x.numel() // cols, cols, cols


def _apply(x, drop, seed, offset, offset_t):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x, rows, cols, stride = _rows(x)
    with on_device(x.device):
        rc = _lib.lib().rnnt_mi355x_dropout(x.data_ptr(), stride, y.data_ptr(), rows, cols, dtype_code("dropout", x), drop, seed, offset,
                                            None if offset_t is None else offset_t.data_ptr(), stream(x.device))
    check(rc, "rnnt_mi355x_dropout")
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, drop, seed, offset, offset_t):
        ctx.args = (drop, seed, offset)
        ctx.save_for_backward(offset_t)  # its version is checked: the backward pass needs the same offset
        return _apply(x, drop, seed, offset, offset_t)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (offset_t,) = ctx.saved_tensors
        return _apply(dy, *ctx.args, offset_t), None, None, None, None


def dropout(x, rate, seed=0, offset=0):
    """x with elements dropped at `rate` (rounded to steps of 2^-16) and the others scaled by 1 / (1 - rate).

    x: float32, bfloat16 or float16, any shape.  seed: an integer below 2^64.  offset: an integer below 2^64, or one int64
    on the device (read by the kernel: inside a captured graph the caller advances it between replays); calls that need
    independent masks take different offsets.  rate 0 returns x itself."""
    dev = need_gpu("dropout", x=x)
    dtype_code("dropout", x)
    drop = drop16("dropout", rate)
    seed, offset, offset_t = seed_offset("dropout", seed, offset, dev)
    if drop == 0 or x.numel() == 0:
        return x
    if x.dim() == 0:
        return dropout(x.reshape(1), rate, seed, offset if offset_t is None else offset_t).reshape(())
    if not x.requires_grad or not torch.is_grad_enabled():
        return _apply(x, drop, seed, offset, offset_t)
    return _DropoutFn.apply(x, drop, seed, offset, offset_t)
