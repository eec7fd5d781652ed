"""Dense layer of any width with bias, activation, dropout and residual in the product's epilogue, and its backward pass.

One TimeDistributed(Dense) with the Dropout behind it, as get_fc stacks them (reference rnnt/keras_model.py:83-104), in
float32, bfloat16 or float16 and at any size: the joint's layers over a training batch, and the same layers on a decoder's
few rows.  ``joint_dense`` is the float32 form for widths up to 128 and keeps its kernels.
"""
from __future__ import annotations

from . import _lib
from ._operator import drop16, seed_offset

ACTIVATIONS = {"linear": 0, "tanh": 1, "relu": 2, "gelu": 3, "silu": 4}


def dense(x, kernel, bias=None, activation="linear", residual=None, dropout=0.0, seed=0, offset=0):
    """residual + dropout(activation(x @ kernel + bias)), differentiable in x, kernel, bias and residual.

    x [..., in], kernel [in, out] (Keras layout), bias [out], residual [..., out]: one of float32, bfloat16, float16, the same
    for all; the result has that type.  Products of float32 inputs are float32's, and sums are float32 throughout.  activation:
    "linear", "tanh", "relu", "gelu" (z times the normal distribution's function) or "silu", with errors relative to the
    result, below 2^-17 of it in float32 up to |z| = 5.  In 16 bits the gradient of the pre-activation is rounded to the type before its
    two products, as the result is before it leaves.  dropout, seed, offset: as ``rnnt_amd.dropout`` takes them, the mask being the
    one it draws for the result; rate 0 at inference.

    The same inputs give the same bits, forward and backward.  The gradient is not differentiable itself (create_graph is
    refused), and forward-mode differentiation is refused."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"dense: activation must be one of {', '.join(ACTIVATIONS)}")
    drop = drop16("dense", dropout) if dropout else 0
    if not drop:
        return _lib.native().dense(x, kernel, bias, residual, act, 0, 0, 0, None)
    return _lib.native().dense(x, kernel, bias, residual, act, drop, *seed_offset("dense", seed, offset, x.device))
