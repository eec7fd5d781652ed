"""Dropout with a counter-based mask that is never stored (the Dropout layers of reference rnnt/keras_model.py:102-103).

The mask is a function of (seed, offset, row, column) alone: the backward pass draws it again, and so can any other code
(``dense`` draws the same one in its epilogue).  Element (r, c) of x seen as [rows, last dimension] takes 16 bits of
Philox4x32-10 at counter (c // 8, r, offset) under the key seed; it is kept when they are >= round(rate * 65536) and then
multiplied by 65536 / (65536 - round(rate * 65536)).  A dropped infinity or NaN becomes 0.
"""
from __future__ import annotations

import torch

from . import _lib
from ._operator import drop16, seed_offset


def dropout(x, rate, seed=0, offset=0):
    """x with elements dropped at `rate` (rounded to steps of 2^-16) and the others scaled by 1 / (1 - rate).

    x: float32, bfloat16 or float16, any shape whose last dimension is below 2^31.  seed: an integer below 2^64.  offset: an integer below 2^64, or one int64
    on the device (read by the kernel: inside a captured graph the caller advances it between replays); calls that need
    independent masks take different offsets.  rate 0 returns x itself.  Differentiable any number of times, backward; forward-mode
    differentiation is refused."""
    native = _lib.native()
    if not isinstance(x, torch.Tensor):
        raise TypeError("dropout: x must be a tensor")
    drop = drop16("dropout", rate)
    seed, offset, offset_t = seed_offset("dropout", seed, offset, x.device)
    if x.dim() == 0:
        return native.dropout(x.reshape(1), drop, seed, offset, offset_t).reshape(())
    return native.dropout(x, drop, seed, offset, offset_t)
