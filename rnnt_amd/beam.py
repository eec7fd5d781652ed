"""One step of a beam search on the MI355X: selection over beams x vocabulary, and the states in their new order.

``KerasRNNTDecoder.beam_search`` (reference rnnt/rnnt_decoder.py:95-233) adds a hypothesis's score to the log-probabilities
of its inner step and keeps the best candidates, one hypothesis at a time on the host.  ``beam_select`` does a whole batch
of beams in one or two launches straight from the joint's logits (log-softmax included, see also ``joint_log_softmax``);
``beam_reorder`` gathers every state tensor of the hypotheses in one more.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._operator import check, dtype_code, need_gpu, on_device, stream

MAX_BEAMS = 64
_INT = 0x7FFFFFFF  # sizes the C entry points take as int
MAX_WIDTH = 64


def beam_select(logits, scores, width, enc=None, allowed=None, finished=None, end=0):
    """The `width` best continuations of every utterance's beams.

    logits [B, K, V] (float32, bfloat16 or float16): the joint's output for K hypotheses, or, with enc [B, V] of the same
    type, the prediction network's part of an additive joint (logits + enc, rounded to float32, as joint_log_softmax does).
    scores [B, K] float32: log-probabilities so far; -inf, NaN or anything beyond +-2^30 marks an empty beam.
    allowed: bool [V] or [B, V]; a forbidden symbol is no candidate and has no part in the softmax, whatever its logit.
    finished: bool [B, K]; such a beam is carried along, as one candidate with its own score at symbol `end`, allowed or not (in
    a transducer: a hypothesis that has emitted blank and waits for the next frame).  Nothing is differentiable here.

    Returns scores [B, width] float32, parent [B, width] int32 (beam) and token [B, width] int32, in descending order of
    scores + log_softmax (compared in float64), ties to the lowest beam, then the lowest symbol.  Where there are fewer
    candidates than `width`: -inf, -1, -1.  A beam whose allowed logits hold NaN or +inf, or nothing above -inf, has none."""
    dev = need_gpu("beam_select", logits=logits, scores=scores, enc=enc, allowed=allowed, finished=finished)
    code = dtype_code("beam_select", logits)
    if logits.dim() != 3 or logits.numel() == 0:
        raise ValueError(f"beam_select: expected logits[B,K,V], got {tuple(logits.shape)}")
    B, K, V = logits.shape
    width = int(width)
    if not 1 <= width <= MAX_WIDTH or K > MAX_BEAMS:
        raise ValueError(f"beam_select: 1 to {MAX_WIDTH} continuations of at most {MAX_BEAMS} beams, got {width} of {K}")
    if K * V > _INT or B > _INT:
        raise ValueError(f"beam_select: beams x vocabulary must stay below 2^31, got {tuple(logits.shape)}")
    if scores.shape != (B, K) or scores.dtype != torch.float32:
        raise ValueError("beam_select: scores must be float32 [B, K]")
    if enc is not None and (enc.shape != (B, V) or enc.dtype != logits.dtype):
        raise ValueError("beam_select: enc must be [B, V] of the logits' type")
    if allowed is not None and (allowed.dtype != torch.bool or allowed.shape not in ((V,), (B, V))):
        raise ValueError("beam_select: allowed must be bool [V] or [B, V]")
    if finished is not None:
        if finished.dtype != torch.bool or finished.shape != (B, K):
            raise ValueError("beam_select: finished must be bool [B, K]")
        if not 0 <= int(end) < V:
            raise ValueError(f"beam_select: end {end} outside [0, {V})")
    s0, s1, s2 = logits.stride()
    if s2 != 1 and V > 1:
        logits = logits.contiguous()
        s0, s1, s2 = logits.stride()
    enc_p = enc_s = allowed_p = allowed_s = fin_p = ws_p = 0
    if enc is not None:
        if V > 1 and enc.stride(1) != 1:
            enc = enc.contiguous()
        enc_p, enc_s = enc.data_ptr(), enc.stride(0)
    if allowed is not None:
        if V > 1 and allowed.stride(-1) != 1:
            allowed = allowed.contiguous()
        allowed_p, allowed_s = allowed.data_ptr(), allowed.stride(0) if allowed.dim() == 2 else 0
    if finished is not None:
        finished = finished.contiguous()
        fin_p = finished.data_ptr()
    scores = scores.contiguous()
    out = torch.empty((3, B, width), dtype=torch.int32, device=dev)
    out_scores, parent, token = out.unbind(0)
    L = _lib.lib()
    with on_device(dev):
        if V > 2048:  # rows of one piece need no workspace
            n = ctypes.c_size_t(0)
            check(L.rnnt_mi355x_beam_select_workspace_bytes(B, K, V, width, ctypes.byref(n)), "rnnt_mi355x_beam_select_workspace_bytes")
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
            ws_p = ws.data_ptr()
        o, step = out.data_ptr(), 4 * B * width
        rc = L.rnnt_mi355x_beam_select(logits.data_ptr(), s0, s1, code, enc_p, enc_s, scores.data_ptr(), allowed_p, allowed_s, fin_p,
                                       int(end) if fin_p else 0, B, K, V, width, o, o + step, o + 2 * step, ws_p, stream(dev))
    if rc:
        check(rc, "rnnt_mi355x_beam_select")
    return out_scores.view(torch.float32), parent, token


def _bytes_of(t):
    """(first, one past the last) byte address a tensor covers."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def beam_reorder(parent, states, batch_dim=0, out=None):
    """Network states, token histories, lengths ... of the hypotheses beam_select kept.

    parent: int32 [B, W] as beam_select returns it.  states: a list of tensors of any type whose dimensions batch_dim and
    batch_dim + 1 are (B, K) -- [layers, B, K, hidden] has batch_dim 1.  Returns a list with W in the place of K and row
    parent[b, w] of utterance b at [b, w]; zeros where parent is -1 (any value outside [0, K)).  out: tensors to write to
    instead of new ones, dense, of the results' shapes and types, sharing no memory with states or one another."""
    if not isinstance(parent, torch.Tensor) or parent.dtype != torch.int32 or parent.dim() != 2:
        raise ValueError("beam_reorder: parent must be int32 [B, W]")
    states = list(states)
    dev = need_gpu("beam_reorder", parent=parent)
    if any(not isinstance(s, torch.Tensor) or s.device != dev for s in states):
        need_gpu("beam_reorder", parent=parent, **{f"states[{i}]": s for i, s in enumerate(states)})
    B, W = parent.shape
    d = int(batch_dim)
    if d < 0:
        raise ValueError("beam_reorder: batch_dim counts from the first dimension")
    K = -1
    new = []
    for i, s in enumerate(states):
        shape = s.shape
        if len(shape) < d + 2 or shape[d] != B:
            raise ValueError(f"beam_reorder: states[{i}] has shape {tuple(shape)}, expected B={B} at dimension {d} and the beams next")
        if K < 0:
            K = shape[d + 1]
        elif shape[d + 1] != K:
            raise ValueError("beam_reorder: the states differ in their number of beams")
        new.append((*shape[:d + 1], W, *shape[d + 2:]))
    if out is None:
        out = [torch.empty(shape, dtype=s.dtype, device=dev) for s, shape in zip(states, new)]
    else:
        out = list(out)
        need_gpu("beam_reorder", parent=parent, **{f"out[{i}]": o for i, o in enumerate(out)})
        if len(out) != len(states) or any(o.shape != sh or o.dtype != s.dtype or not o.is_contiguous() for o, s, sh in zip(out, states, new)):
            raise ValueError("beam_reorder: out must be dense tensors of the results' shapes and types")
        spans = [(*_bytes_of(t), i < len(out)) for i, t in enumerate([*out, *states, parent]) if t.numel()]
        for i, (a0, a1, written) in enumerate(spans):
            if written and any(a0 < b1 and b0 < a1 for j, (b0, b1, _) in enumerate(spans) if j != i):
                raise ValueError("beam_reorder: out overlaps a state, another output or parent")
    if max(B, K, W) > _INT:
        raise ValueError("beam_reorder: more than 2^31 - 1 utterances or beams")
    if K == 0:
        for o in out:
            o.zero_()
        return out
    if not parent.is_contiguous():
        parent = parent.contiguous()
    table, keep = [], []  # the fields of rnnt_mi355x_reorder_tensor, one tensor after the other
    for s, o in zip(states, out):
        n = o.numel()
        if n == 0:
            continue
        # [outer, B, K, row]: the row has to be dense, the three leading dimensions need one stride each
        if not s.is_contiguous() and (d > 1 or not s[(0,) * (d + 2)].is_contiguous()):
            s = s.contiguous()
            keep.append(s)
        e, strides = s.element_size(), s.stride()
        outer = s.shape[0] if d == 1 else math.prod(s.shape[:d])
        table += (s.data_ptr(), o.data_ptr(), outer, strides[d - 1] * e if d else 0, strides[d] * e, strides[d + 1] * e, n // (outer * B * W) * e)
    f, most = _lib.lib().rnnt_mi355x_beam_reorder, 7 * _lib.REORDER_MAX
    with on_device(dev):
        for i in range(0, len(table), most):
            part = table[i:i + most]
            rc = f((ctypes.c_longlong * len(part))(*part), len(part) // 7, parent.data_ptr(), B, K, W, stream(dev))
            if rc:
                check(rc, "rnnt_mi355x_beam_reorder")
    return out
