"""Dropout with a counter-based mask that is never stored (the Dropout layers of reference rnnt/keras_model.py:102-103).

The mask is a function of (seed, offset, row, column) alone: the backward pass draws it again, and so can any other code
(``dense`` draws the same one in its epilogue).  Element (r, c) of x seen as [rows, last dimension] takes 16 bits of
Philox4x32-10 at counter (c // 8, r, offset) under the key seed; it is kept when they are >= round(rate * 65536) and then
multiplied by 65536 / (65536 - round(rate * 65536)).  A dropped infinity or NaN becomes 0.
"""
from __future__ import annotations

import torch

from . import _lib
from ._operator import DTYPE_CODE, check, drop16, dtype_code, need_gpu, on_device, seed_offset, stream


def _apply(x, drop, seed, offset, offset_t):
    cols = stride = x.shape[-1]
    if cols > 0x7FFFFFFF:  # the C entry point takes it as an int
        raise ValueError("dropout: the last dimension holds 2^31 elements or more")
    if x.is_contiguous():
        y = torch.empty_like(x)
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        # rows of a matrix may be any distance apart; anything else is made dense
        if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= cols:
            stride = x.stride(0)
        else:
            x = x.contiguous()
    dev = x.device
    with on_device(dev):
        rc = _lib.lib().rnnt_mi355x_dropout(x.data_ptr(), stride, y.data_ptr(), x.numel() // cols, cols, DTYPE_CODE[x.dtype], drop, seed, offset,
                                            None if offset_t is None else offset_t.data_ptr(), stream(dev))
    if rc:
        check(rc, "rnnt_mi355x_dropout")
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, drop, seed, offset, offset_t):
        ctx.args = (drop, seed, offset)
        if offset_t is not None:
            ctx.save_for_backward(offset_t)  # its version is checked: the backward pass needs the same offset
        ctx.has_offset = offset_t is not None
        return _apply(x, drop, seed, offset, offset_t)

    @staticmethod
    def backward(ctx, dy):
        args = (*ctx.args, ctx.saved_tensors[0] if ctx.has_offset else None)
        if torch.is_grad_enabled():  # a graph of the gradient is wanted: the same linear map again
            return _DropoutFn.apply(dy, *args), None, None, None, None
        return _apply(dy, *args), None, None, None, None


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
