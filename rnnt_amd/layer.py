"""Dense layer of any width with bias, activation, dropout and residual in the product's epilogue, and its backward pass.

One TimeDistributed(Dense) with the Dropout behind it, as get_fc stacks them (reference rnnt/keras_model.py:83-104), in
float32, bfloat16 or float16 and at any size: the joint's layers over a training batch, and the same layers on a decoder's
few rows.  ``joint_dense`` is the float32 form for widths up to 128 and keeps its kernels.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._operator import DTYPE_CODE, check, drop16, dtype_code, need_gpu, on_device, seed_offset, stream

ACTIVATIONS = {"linear": 0, "tanh": 1, "relu": 2, "gelu": 3, "silu": 4}
MAX_WIDTH = 1 << 24  # inputs and outputs of rnnt_mi355x_layer_*
_AUX_TYPE = {torch.float32: torch.float32, torch.bfloat16: torch.float16, torch.float16: torch.float32}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _as_rows(t):
    """t as [rows, last dimension] whose last dimension is contiguous: (tensor, row stride)."""
    n = t.shape[-1]
    if t.is_contiguous():
        return (t if t.dim() == 2 else t.view(-1, n)), n
    if t.dim() != 2:
        t = t.reshape(-1, n)
    if (n > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < n):
        t = t.contiguous()
    return t, max(t.stride(0), n) if t.shape[0] > 1 else n


def _layer(x, x_stride, kernel, kernel_stride, bias, residual, residual_stride, y, aux, act, drop, seed, offset, offset_t):
    n_in, n_out = kernel.shape
    # positional: the order of rnnt_mi355x_layer
    return _lib.Layer(x.data_ptr(), kernel.data_ptr(), _ptr(bias), _ptr(residual), _ptr(y), _ptr(aux), x_stride, kernel_stride, residual_stride,
                      x.shape[0], n_in, n_out, DTYPE_CODE[x.dtype], act, drop, seed, offset, _ptr(offset_t))


def _forward(x, kernel, bias, residual, act, drop, seed, offset, offset_t, want_aux):
    """(y, aux or None)"""
    dev, shape = x.device, (*x.shape[:-1], kernel.shape[1])
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    aux = torch.empty(shape, dtype=_AUX_TYPE[x.dtype], device=dev) if want_aux else None
    if y.numel() == 0:
        return y, aux
    x, x_stride = _as_rows(x)
    kernel, kernel_stride = _as_rows(kernel)
    residual_stride, ws_p = 0, None
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if residual is not None:
        residual, residual_stride = _as_rows(residual)
    layer = ctypes.byref(_layer(x, x_stride, kernel, kernel_stride, bias, residual, residual_stride, y, aux, act, drop, seed, offset, offset_t))
    L = _lib.lib()
    with on_device(dev):
        n = ctypes.c_size_t(0)
        rc = L.rnnt_mi355x_layer_workspace_bytes(layer, None, 0, ctypes.byref(n), None)
        if n.value:
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
            ws_p = ws.data_ptr()
        rc = rc or L.rnnt_mi355x_layer_forward(layer, ws_p, stream(dev))
    if rc:
        check(rc, "rnnt_mi355x_layer_forward")
    return y, aux


class _LayerFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, residual, act, drop, seed, offset, offset_t):
        # what act' is computed from: the pre-activation, or the output where that is as good
        from_y = residual is None and (act == 2 or (act == 1 and x.dtype == torch.float32))
        want_aux = act != 0 and not from_y and any(ctx.needs_input_grad[:3])
        y, aux = _forward(x, kernel, bias, residual, act, drop, seed, offset, offset_t, want_aux)
        ctx.save_for_backward(x, kernel, y if act != 0 and from_y else None, aux, offset_t)
        ctx.args = (act, drop, seed, offset)
        ctx.n_bias = None if bias is None else bias.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("dense: the gradient is not differentiable (create_graph)")
        x, kernel, y, aux, offset_t = ctx.saved_tensors
        need_x, need_k, need_b, need_r = ctx.needs_input_grad[:4]
        d_residual = dy if need_r else None
        if not (need_x or need_k or need_b):
            return (None, None, None, d_residual) + (None,) * 5
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dk = torch.empty(kernel.shape, dtype=x.dtype, device=x.device) if need_k else None
        db = torch.empty(ctx.n_bias, dtype=x.dtype, device=x.device) if need_b else None
        if dy.numel() == 0:
            return tuple(None if t is None else t.zero_() for t in (dx, dk, db)) + (d_residual,) + (None,) * 5
        x, x_stride = _as_rows(x)
        kernel, kernel_stride = _as_rows(kernel)
        dy, dy_stride = _as_rows(dy)
        dev, dy_p = x.device, dy.data_ptr()
        layer = ctypes.byref(_layer(x, x_stride, kernel, kernel_stride, None, None, 0, y, aux, *ctx.args, offset_t))
        L = _lib.lib()
        with on_device(dev):
            n = ctypes.c_size_t(0)
            rc = L.rnnt_mi355x_layer_workspace_bytes(layer, dy_p, dy_stride, None, ctypes.byref(n))
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
            rc = rc or L.rnnt_mi355x_layer_backward(layer, dy_p, dy_stride, _ptr(dx), _ptr(dk), _ptr(db), ws.data_ptr(), stream(dev))
        if rc:
            check(rc, "rnnt_mi355x_layer_backward")
        return (dx, dk, db, d_residual) + (None,) * 5


def dense(x, kernel, bias=None, activation="linear", residual=None, dropout=0.0, seed=0, offset=0):
    """residual + dropout(activation(x @ kernel + bias)), differentiable in x, kernel, bias and residual.

    x [..., in], kernel [in, out] (Keras layout), bias [out], residual [..., out]: one of float32, bfloat16, float16, the same
    for all; the result has that type, products and sums are float32 throughout (float32 inputs included).  activation:
    "linear", "tanh", "relu", "gelu" (z times the normal distribution's function) or "silu".  dropout, seed, offset: as
    ``rnnt_amd.dropout`` takes them, the mask being the one it draws for the result; rate 0 at inference.

    The same inputs give the same bits, forward and backward."""
    dev = need_gpu("dense", x=x, kernel=kernel, bias=bias, residual=residual)
    dtype_code("dense", x)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"dense: activation must be one of {', '.join(ACTIVATIONS)}")
    if kernel.dim() != 2 or x.dim() < 1 or x.shape[-1] != kernel.shape[0] or 0 in kernel.shape:
        raise ValueError(f"dense: x{tuple(x.shape)} does not fit kernel{tuple(kernel.shape)}")
    if max(kernel.shape) > MAX_WIDTH:
        raise ValueError(f"dense: a layer is at most {MAX_WIDTH} wide, got kernel{tuple(kernel.shape)}")
    if bias is not None and bias.shape != kernel.shape[1:]:
        raise ValueError(f"dense: bias{tuple(bias.shape)} does not fit kernel{tuple(kernel.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + kernel.shape[1:]:
        raise ValueError(f"dense: residual{tuple(residual.shape)} is not of the result's shape")
    for name, t in (("kernel", kernel), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"dense: {name} is {t.dtype}, x is {x.dtype}")
    drop = drop16("dense", dropout)
    seed, offset, offset_t = seed_offset("dense", seed, offset, dev) if drop else (0, 0, None)
    if torch.is_grad_enabled() and (x.requires_grad or kernel.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LayerFn.apply(x, kernel, bias, residual, act, drop, seed, offset, offset_t)
    return _forward(x, kernel, bias, residual, act, drop, seed, offset, offset_t, False)[0]
