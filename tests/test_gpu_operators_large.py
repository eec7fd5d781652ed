"""Tensors of more than 2^31 elements: what lies behind has to be what a small call gives for it."""
import numpy as np
import pytest
import torch

import rnnt_amd
from oracle import operators as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_dense_result_beyond_2_31():
    M, K, N = 270_000, 24, 8192
    x = torch.randn(M, K, device=DEV).bfloat16()
    w = torch.randn(K, N, device=DEV).bfloat16().requires_grad_(True)
    b = torch.randn(N, device=DEV).bfloat16()
    y = rnnt_amd.dense(x, w, b, "silu", dropout=0.5, seed=1, offset=2)
    tail = slice(M - 3, M)
    z = x[tail].double() @ w.detach().double() + b.double()
    c = [np.full(N // 8, v, np.uint64) for v in (0, 0, 2, 0)]
    c[0] = np.arange(N // 8, dtype=np.uint64)
    for i in range(3):
        c[1] = np.full(N // 8, M - 3 + i, np.uint64)
        u = np.stack([h for q in orc.philox4x32(c, (1, 0)) for h in (q & np.uint64(0xFFFF), q >> np.uint64(16))], axis=1).reshape(N)
        want = z[i] * torch.sigmoid(z[i]) * torch.from_numpy((u >= 32768) * 2.0).to(DEV)
        # K = 24 products (24 * 2^-24 of some 20) and the formula, both under 2^-16; a rounding to bfloat16
        assert ((y[M - 3 + i].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15).all()
    # the kernel's gradient: all of dy but the last row is zero
    dy = torch.zeros_like(y)
    dy[M - 1] = 1
    (dw,) = torch.autograd.grad(y, w, dy)
    p = torch.sigmoid(z[2])
    dz = (p * (1 + z[2] * (1 - p)) * torch.from_numpy((u >= 32768) * 2.0).to(DEV)).bfloat16().double()
    want = x[M - 1].double().unsqueeze(1) * dz.unsqueeze(0)
    # dz may be rounded the other way (2^-7 of itself), its slope comes from a float16 pre-activation (2^-11 |z|, |act''| < 1, doubled by
    # the dropout's scale), dw is rounded once
    tol = 2.0 ** -7 * want.abs() * 1.5 + x[M - 1].double().abs().unsqueeze(1) * (2.0 ** -10 * z[2].abs() + 2.0 ** -18)
    assert ((dw.double() - want).abs() <= tol).all()


def test_dropout_beyond_2_31():
    rows, cols = 70_000, 32_768
    y = rnnt_amd.dropout(torch.ones(rows, cols, device=DEV, dtype=torch.float16), 0.25, seed=3, offset=4)
    c = [np.arange(cols // 8, dtype=np.uint64), np.full(cols // 8, rows - 1, np.uint64), np.full(cols // 8, 4, np.uint64), np.zeros(cols // 8, np.uint64)]
    u = np.stack([h for q in orc.philox4x32(c, (3, 0)) for h in (q & np.uint64(0xFFFF), q >> np.uint64(16))], axis=1).reshape(cols)
    assert ((y[-1] > 0).cpu().numpy() == (u >= 16384)).all()


def test_beam_logits_beyond_2_31_elements():
    B, K, V = 36, 32, 1_900_001
    logits = torch.empty(B, K, V, device=DEV, dtype=torch.bfloat16).normal_()
    scores = torch.rand(B, K, device=DEV) * -3
    got = rnnt_amd.beam_select(logits, scores, 16)
    for b in (0, B - 1):
        one = rnnt_amd.beam_select(logits[b:b + 1].clone(), scores[b:b + 1].clone(), 16)
        assert all(torch.equal(g[b], o[0]) for g, o in zip(got, one))
    best = scores[-1].double() + (logits[-1].double() - torch.logsumexp(logits[-1].double(), dim=1, keepdim=True)).amax(dim=1)
    assert abs(best.max().item() - got[0][-1, 0].item()) < 2.0 ** -20


def test_reorder_beyond_2_31_bytes():
    states = torch.arange(40 * 4, device=DEV, dtype=torch.int32).view(40, 4, 1).expand(40, 4, 4_000_000).contiguous()
    parent = torch.randint(0, 4, (40, 4), device=DEV, dtype=torch.int32)
    (out,) = rnnt_amd.beam_reorder(parent, [states])
    want = torch.arange(40, device=DEV).unsqueeze(1) * 4 + parent
    assert torch.equal(out[:, :, 0].long(), want.long()) and torch.equal(out[:, :, -1].long(), want.long())


def test_reorder_of_more_rows_than_a_launch_has_wavefronts():
    """2^26 rows and some, a wavefront each: a launch holds fewer than 2^32 threads."""
    B, K, W = (1 << 20) + 3, 5, 64
    states = torch.randint(0, 256, (B, K), device=DEV, dtype=torch.uint8)
    parent = torch.randint(-1, K, (B, W), device=DEV, dtype=torch.int32)
    (out,) = rnnt_amd.beam_reorder(parent, [states])
    for part in (slice(0, 1000), slice(B // 2 - 500, B // 2 + 500), slice(B - 1000, B)):
        p = parent[part].long()
        assert torch.equal(out[part], torch.where(p < 0, 0, states[part].gather(1, p.clamp(min=0))))


def test_dropout_of_the_longest_row():
    n = (1 << 31) - 1
    x = torch.ones(n, device=DEV, dtype=torch.float16)
    y = rnnt_amd.dropout(x, 0.25, seed=3, offset=4)
    groups = np.arange((n + 7) // 8 - 4, (n + 7) // 8, dtype=np.uint64)
    c = [groups, np.zeros_like(groups), np.full_like(groups, 4), np.zeros_like(groups)]
    u = np.stack([h for q in orc.philox4x32(c, (3, 0)) for h in (q & np.uint64(0xFFFF), q >> np.uint64(16))], axis=1).reshape(-1)[:31]
    assert ((y[-31:] > 0).cpu().numpy() == (u >= 16384)).all()
