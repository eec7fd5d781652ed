"""Plain float64 numpy forms of the operators around the joint network: the counter-based dropout mask, Dense with its
epilogue, the beam step.  An oracle, like everything in this folder."""
import math

import numpy as np


def philox4x32(c, k, rounds=10):
    """c: four arrays of uint64 words below 2^32; k: (k0, k1) integers.  Philox4x32 of Salmon et al., 2011."""
    m = np.uint64(0xFFFFFFFF)
    c = [np.asarray(w, np.uint64) for w in c]
    k0, k1 = k
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c


def dropout_scale(rows, cols, rate, seed, offset):
    """[rows, cols] float64: 0 where dropped, 1/keep elsewhere."""
    groups = -(-cols // 8)
    g, r = np.meshgrid(np.arange(groups), np.arange(rows))
    w = philox4x32((g, r, np.full_like(g, offset % 2 ** 32), np.full_like(g, offset >> 32)), (seed % 2 ** 32, seed >> 32))
    u = np.stack([h for x in w for h in (x & np.uint64(0xFFFF), x >> np.uint64(16))], axis=-1).reshape(rows, groups * 8)[:, :cols]
    drop = round(rate * 65536)
    return (u >= np.uint64(drop)) * (65536.0 / (65536 - drop))


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(z, name):
    """(act(z), act'(z))"""
    if name == "linear":
        return z, np.ones_like(z)
    if name == "tanh":
        a = np.tanh(z)
        return a, 1 - a * a
    if name == "relu":
        return np.where(z > 0, z, 0.0), (z > 0) * 1.0
    if name == "gelu":
        half = 0.5 * (1 + _erf(z / math.sqrt(2)))
        return z * half, half + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    p = 1 / (1 + np.exp(-z))
    return z * p, p * (1 + z * (1 - p))


def dense(x, kernel, bias=None, act="linear", residual=None, scale=None, dy=None):
    """y, and with dy the gradients (dx, dkernel, dbias); scale: what dropout_scale gives."""
    x, kernel = np.asarray(x, np.float64), np.asarray(kernel, np.float64)
    z = x @ kernel + (0.0 if bias is None else np.asarray(bias, np.float64))
    a, slope = activation(z, act)
    s = 1.0 if scale is None else scale
    y = a * s + (0.0 if residual is None else np.asarray(residual, np.float64))
    if dy is None:
        return y
    dz = np.asarray(dy, np.float64) * s * slope
    return y, dz @ kernel.T, x.T @ dz, dz.sum(axis=0)


def beam_select(logits, scores, width, enc=None, allowed=None, finished=None, end=0):
    """logits [B, K, V], enc [B, V] float32 arrays; returns scores, parent, token [B, width] and the totals of every place."""
    B, K, V = logits.shape
    out = np.full((B, width), -np.inf), np.full((B, width), -1, np.int32), np.full((B, width), -1, np.int32)
    for b in range(B):
        cand = []
        for k in range(K):
            s = float(scores[b, k])
            if not abs(s) <= 2.0 ** 30:
                continue
            if finished is not None and finished[b, k]:
                cand.append((s, k * V + end))
                continue
            x = logits[b, k] if enc is None else (logits[b, k] + enc[b]).astype(np.float32)
            x = x.astype(np.float64)
            if allowed is not None:
                x = np.where(allowed if allowed.ndim == 1 else allowed[b], x, -np.inf)
            if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
                continue
            m = x.max()
            t = s + ((x - m) - math.log(np.exp(x - m).sum()))
            cand += [(float(t[v]), k * V + v) for v in np.nonzero(x > -np.inf)[0]]
        cand.sort(key=lambda c: (-c[0], c[1]))
        for i, (t, flat) in enumerate(cand[:width]):
            out[0][b, i], out[1][b, i], out[2][b, i] = t, flat // V, flat % V
    return out
