"""Dense layer with its epilogue against the float64 oracle.

Tolerances, with u = half a step of the type (fp32 2^-24, bf16 2^-8, fp16 2^-11; float16 below 2^-14: 2^-25 absolute):
  product       a float32 accumulation of K products: each of at most K + 3 roundings is 2^-24 of a partial sum, which is
                bounded by S = sum |a||b|; with K = 5000 that bound is 3e-4 S, while the roundings are independent and grow as
                sqrt(K).  8 sqrt(K + 8) 2^-24 S is taken for z (eight standard deviations).
  activation    |act'| <= 1.13, so z's error passes on by that, plus 2^-21 (1 + |z|) of the activation's own formula; gelu in 16
                bits has a Phi(z) that is off by up to 1.5e-6 < 2^-19.3, so up to 2^-19.3 |z|, next to a rounding of 2^-11 |z| / 2
  dropout       the scale 1/keep multiplies all of it, and adds its rounding
  result        u |y| for the rounding of y
  gradients     dz carries act' (2^-20 of itself; the saved pre-activation of a bf16 layer is float16: 2^-11 |z| and |act''| <= 0.8;
                a float32 one has the product's own error) and one rounding u to the type; dx, dkernel, dbias then are sums
                of such terms: the same bound with S over |dz||w| plus the sum of the terms' errors.
"""
import math

import numpy as np
import pytest
import torch

import rnnt_amd
from oracle import operators as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def data(M, K, N, dtype, seed, bias=True, residual=False):
    g = torch.Generator().manual_seed(seed)
    def t(*s, scale=1.0):
        return (torch.randn(s, generator=g) * scale).to(dtype)
    return t(M, K), t(K, N, scale=K ** -0.5), t(N) if bias else None, t(M, N) if residual else None, t(M, N)


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def acc(k, s):
    return 8 * np.sqrt(k + 8.0) * 2.0 ** -24 * s


def check_layer(M, K, N, dtype, act="linear", bias=True, residual=False, rate=0.0, seed=1, tensors=None):
    x, w, b, r, dy = tensors or data(M, K, N, dtype, seed, bias, residual)
    kw = dict(activation=act, dropout=rate, seed=77, offset=2 ** 33 + 5)
    leaves = [None if t is None else t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
    y = rnnt_amd.dense(leaves[0], leaves[1], leaves[2], residual=leaves[3], **kw)
    with torch.no_grad():
        assert torch.equal(y, rnnt_amd.dense(leaves[0], leaves[1], leaves[2], residual=leaves[3], **kw))
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(DEV))
    X, W, Bv, R, DY = map(f64, (x, w, b, r, dy))
    scale = orc.dropout_scale(M, N, rate, 77, 2 ** 33 + 5) if rate else np.ones((M, N))
    want = orc.dense(X, W, Bv, act, R, scale, DY)
    u, least = U[dtype], LEAST[dtype]
    z = X @ W + (0 if Bv is None else Bv)
    sz = np.abs(X) @ np.abs(W) + (0 if Bv is None else np.abs(Bv))
    ez = acc(K, sz)
    formula = 0 if act == "linear" else (2.0 ** -21 if act != "gelu" or dtype == torch.float32 else 2.0 ** -19) * (1 + np.abs(z))
    ey = scale * (1.13 * ez + formula + 2.0 ** -22 * np.abs(z)) + 2.0 ** -24 * np.abs(want[0])
    tol = ey + np.maximum(u * (np.abs(want[0]) + ey), least)
    got = f64(y)
    bad = np.abs(got - want[0]) > tol
    assert not bad.any(), (np.abs(got - want[0])[bad][:4], tol[bad][:4], np.argwhere(bad)[:4], bad.sum())
    dz = DY * scale * orc.activation(z, act)[1]
    if act == "linear":
        esl = np.zeros_like(z)
    elif act == "relu":
        esl = (np.abs(z) <= ez) * 1.0  # next to the border either slope is right
    else:
        esl = 2.0 ** -20 * (1 + np.abs(z)) + 0.8 * (ez + (2.0 ** -11 * np.abs(z) + 2.0 ** -24 if dtype == torch.bfloat16 else 0))
        if act == "tanh" and dtype == torch.float32 and r is None:
            esl = esl + 2.0 ** -21  # 1 - y^2 from the rounded y
    edz = np.abs(DY) * scale * esl
    edz = edz + (0 if act == "linear" and not rate else np.maximum(u * (np.abs(dz) + edz), least) + 2.0 ** -22 * np.abs(dz))
    adz = np.abs(dz) + edz
    got = [f64(t) for t in grads]
    for name, g, want_g, s, e, n in (("dx", got[0], want[1], adz @ np.abs(W).T, edz @ np.abs(W).T, N),
                                     ("dkernel", got[1], want[2], np.abs(X).T @ adz, np.abs(X).T @ edz, M)):
        t = acc(n, s) + e
        t = t + np.maximum(u * (np.abs(want_g) + t), least)
        bad = np.abs(g - want_g) > t
        assert not bad.any(), (name, np.abs(g - want_g)[bad][:4], t[bad][:4], np.argwhere(bad)[:4], bad.sum())
    if b is not None:
        t = acc(M, adz.sum(0)) + edz.sum(0)
        t = t + np.maximum(u * (np.abs(want[3]) + t), least)
        assert (np.abs(got[2] - want[3]) <= t).all()
    if r is not None:
        assert torch.equal(grads[-1].cpu(), dy)


SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (8, 250, 62), (31, 33, 40), (32, 64, 128), (33, 64, 72), (64, 520, 136), (65, 129, 66),
          (100, 1000, 65), (130, 96, 130), (257, 72, 264), (300, 515, 103), (129, 2056, 136), (1000, 40, 250),
          (600, 515, 1030), (513, 77, 33), (520, 64, 65), (777, 1003, 130),
          (24, 2100, 2100), (64, 1500, 2056), (33, 100, 4096), (20, 1032, 2048)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_sizes(M, K, N, dtype):
    check_layer(M, K, N, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["linear", "tanh", "relu", "gelu", "silu"])
@pytest.mark.parametrize("residual,rate,bias", [(False, 0.0, False), (False, 0.25, True), (True, 0.0, True), (True, 0.4, False)])
def test_epilogues(act, residual, rate, bias, dtype):
    check_layer(70, 136, 72, dtype, act, bias, residual, rate)
    check_layer(45, 37, 51, dtype, act, bias, residual, rate)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_blocks(dtype):
    """Enough of the result for the largest block, ragged at both ends, with the epilogue."""
    check_layer(3500, 200, 3336, dtype, "gelu", True, False, 0.1)
    check_layer(3331, 136, 3400, dtype, "linear", True, True, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_sums_are_split_and_joined(dtype):
    check_layer(5, 6000, 80, dtype, "silu", True, True, 0.2)  # few rows, long k
    check_layer(9000, 24, 40, dtype, "tanh", True, False, 0.2)  # the kernel gradient's k is the number of rows
    check_layer(7003, 65, 9, dtype, "linear", True, False, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignments(dtype):
    g = torch.Generator().manual_seed(3)
    big = torch.randn(90, 400, generator=g).to(dtype).to(DEV)
    wide = (torch.randn(400, 300, generator=g) * 0.1).to(dtype).to(DEV)
    for x in (big[:, 8:136], big[:, 3:131], big[::3, :128], big.t()[:128, :].t(), big[:, 0:256:2]):
        for w in (wide[:128, 16:112], wide[:128, 5:101], wide[5:133, :96], wide.t()[:96, :128].t()):
            res = big[:x.shape[0], 200:296]
            def run(x, w, res):
                a, b, c = x.detach().requires_grad_(True), w.detach().requires_grad_(True), res.detach().requires_grad_(True)
                y = rnnt_amd.dense(a, b, None, "gelu", c, 0.1, 5, 6)
                up = torch.linspace(-1, 1, y.numel(), device=DEV).to(dtype).view(y.shape[1], y.shape[0]).t()  # an upstream gradient of another layout
                return (y, *torch.autograd.grad(y, (a, b, c), up))
            got, ref = run(x, w, res), run(x.contiguous(), w.contiguous(), res.contiguous())
            for p, q in zip(got, ref):
                # the same products, perhaps along another path of loads: equal but for the order of sums
                assert ((p.float() - q.float()).abs() <= 2 * U[dtype] * q.float().abs() + 2e-5).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_leading_dimensions_and_empty_batches(dtype):
    x, w, b, r, dy = (t.to(DEV) if t is not None else None for t in data(24, 16, 10, dtype, 4, residual=True))
    y = rnnt_amd.dense(x.reshape(2, 3, 4, 16), w, b, "tanh", r.reshape(2, 3, 4, 10), 0.3, 1, 2)
    assert y.shape == (2, 3, 4, 10) and torch.equal(y.reshape(24, 10), rnnt_amd.dense(x, w, b, "tanh", r, 0.3, 1, 2))
    assert torch.equal(rnnt_amd.dense(x[0], w, b), rnnt_amd.dense(x[:1], w, b)[0])
    e = x[:0].requires_grad_(True)
    wg, bg = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    out = rnnt_amd.dense(e, wg, bg, "gelu")
    out.sum().backward()
    assert out.shape == (0, 10) and e.grad.shape == (0, 16) and not wg.grad.any() and not bg.grad.any()


def test_mask_is_the_one_dropout_draws():
    x, w, b, _, _ = (t.to(DEV) if t is not None else None for t in data(130, 40, 77, torch.float32, 5))
    a = rnnt_amd.dense(x, w, b, "tanh", dropout=0.35, seed=9, offset=10)
    assert torch.equal(a, rnnt_amd.dropout(rnnt_amd.dense(x, w, b, "tanh"), 0.35, seed=9, offset=10))


@pytest.mark.parametrize("shape", [(40, 24, 72), (300, 160, 200), (20, 3000, 24)])
def test_infinities_overflow_and_nan(shape):
    """float32 products are made of bfloat16 parts: what those cannot hold has to come out as float32 gives it."""
    M, K, N = shape
    x, w, _, _, _ = data(M, K, N, torch.float32, 6)
    x[1, 2], x[2, 3], x[3, 1], x[4, 0] = float("inf"), float("-inf"), float("nan"), 3.4e38
    w[:, 5] = 0.5
    w[7, 6] = float("inf")
    w[0, :3] = 1.0
    x[5], x[6], w[:, 4] = 1e-38, 1e38, 1e-30
    got = rnnt_amd.dense(x.to(DEV), w.to(DEV)).cpu().double().numpy()
    x, w = x.numpy(), w.numpy()
    with np.errstate(all="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64)
        over = np.abs(want) > 3.4028235e38
    ok = np.isfinite(want) & ~over
    assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    assert np.isfinite(got[ok]).mean() > 0.99  # a finite sum next to float32's end may pass it on the way
    s = np.abs(np.where(np.isfinite(x), x, 0).astype(np.float64)) @ np.abs(np.where(np.isfinite(w), w, 0).astype(np.float64))
    fine = ok & np.isfinite(got)
    # A part of an operand below 2^-126 is subnormal and may count as zero: an operand's parts are each below 2^-8 of the one
    # before, so what is dropped of it is below 2^-126 (1 + 2^-8 + 2^-16), less than 2^-125, times the other operand.
    one = lambda t, axis: np.abs(np.where(np.isfinite(t), t, 0).astype(np.float64)).sum(axis, keepdims=True)  # noqa: E731
    least = 2.0 ** -125 * (one(w, 0) + one(x, 1))
    got, want = got[fine], want[fine]
    assert (np.abs(got - want) <= acc(K, s)[fine] + 2.0 ** -24 * np.abs(want) + least[fine]).all()


def test_everything_nan_ends_soon():
    """A diverged model: every float32 result is computed again, which ends at the first value that is no number."""
    x = torch.full((3000, 20000), float("nan"), device=DEV)
    assert rnnt_amd.dense(x, torch.ones(20000, 300, device=DEV)).isnan().all()


@pytest.mark.parametrize("act", ["tanh", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_far_pre_activations(act, dtype):
    """Values where a formula could overflow: the activation and its slope are at their limits."""
    z = torch.tensor([-3e4, -400.0, -89.0, -30.0, -1e-6, 0.0, 1e-6, 30.0, 89.0, 400.0, 6e4, float("inf"), float("-inf"), float("nan")]).to(dtype)
    x = z.reshape(-1, 1).to(DEV).requires_grad_(True)
    w = torch.ones(1, 1, dtype=dtype, device=DEV)
    y = rnnt_amd.dense(x, w, activation=act, residual=torch.zeros(len(z), 1, dtype=dtype, device=DEV))
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    f = z.double().numpy()
    with np.errstate(all="ignore"):
        a, s = orc.activation(f, act)
    a[-3], a[-2] = {"tanh": (1, -1)}.get(act, (np.inf, 0))
    s[-3], s[-2] = (0, 0) if act == "tanh" else (1, 0)
    got_a, got_s = f64(y)[:, 0], f64(dx)[:, 0]
    a[-1] = s[-1] = 0  # the value that is no number has its own line
    assert np.isnan(got_a[-1]) and (np.isnan(got_s[-1]) or act == "relu")
    assert got_a[-3] == a[-3] and got_a[-2] == a[-2]
    # silu(-400) = -400 e^-400 is no float32: below the smallest normal number, 2^-126, a result may be zero
    f = np.where(np.isfinite(f), f, 0)
    lim = U[dtype] * np.where(np.isfinite(a), np.abs(a), 0) + (2.0 ** -21 if act != "gelu" or dtype == torch.float32 else 2.0 ** -19) * np.maximum(1, np.abs(f)) * (np.abs(f) < 100) + np.maximum(LEAST[dtype], 2.0 ** -126)
    assert (np.abs(got_a[:-3] - a[:-3]) <= lim[:-3]).all()
    assert (np.abs(got_s[:-1] - s[:-1]) <= U[dtype] + 2.0 ** -19 + (2.0 ** -11 if dtype == torch.bfloat16 else 0)).all()


def test_gradients_against_differences():
    x, w, b, r, dy = (t.to(DEV) for t in data(6, 10, 9, torch.float32, 7, residual=True))
    for act in ("tanh", "gelu", "silu"):
        def f(*t):
            return (rnnt_amd.dense(t[0], t[1], t[2], act, t[3], 0.3, 3, 4) * dy).double().sum().item()
        args = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        grads = torch.autograd.grad(rnnt_amd.dense(args[0], args[1], args[2], act, args[3], 0.3, 3, 4), args, dy)
        for i, (t, g) in enumerate(zip((x, w, b, r), grads)):
            for j in (0, t.numel() // 2, t.numel() - 1):
                h, hi, lo = 2.0 ** -6, [q.clone() for q in (x, w, b, r)], [q.clone() for q in (x, w, b, r)]
                hi[i].view(-1)[j] += h
                lo[i].view(-1)[j] -= h
                # central difference: h^2/6 f''' (f''' < 60 here: sums of at most 10 terms |dy| |x|^3 < 4^3 ... / 10) and 54 values'
                # float32 rounding over 2h
                assert abs((f(*hi) - f(*lo)) / (2 * h) - g.view(-1)[j].item()) < h * h * 10 + 54 * 4 * 2.0 ** -23 / (2 * h)


def test_only_the_wanted_gradients():
    x, w, b, r, dy = (t.to(DEV) for t in data(50, 30, 20, torch.float32, 8, residual=True))
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(rnnt_amd.dense(full[0], full[1], full[2], "silu", full[3], 0.2, 1, 1), full, dy)
    for keep in ((0,), (1,), (2,), (3,), (0, 2), (1, 3)):
        t = [q.clone().requires_grad_(i in keep) for i, q in enumerate((x, w, b, r))]
        got = torch.autograd.grad(rnnt_amd.dense(t[0], t[1], t[2], "silu", t[3], 0.2, 1, 1), [t[i] for i in keep], dy)
        assert all(torch.equal(a, want[i]) for a, i in zip(got, keep))


def test_equal_calls_give_equal_bits():
    for dtype in TYPES:
        x, w, b, r, dy = (t.to(DEV) for t in data(5000, 72, 96, dtype, 9, residual=True))
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        runs = []
        for _ in range(3):
            y = rnnt_amd.dense(*leaves, "gelu", r, 0.1, 1, 2)
            runs.append((y, *torch.autograd.grad(y, leaves, dy)))
        for other in runs[1:]:
            assert all(torch.equal(a, c) for a, c in zip(runs[0], other))


def test_streams_and_graphs():
    """Forward and backward captured once, replayed over new inputs and new masks, next to eager work."""
    dtype = torch.bfloat16
    x, w, b, r, dy = (t.to(DEV) for t in data(3000, 64, 48, dtype, 10, residual=True))
    off = torch.zeros(1, dtype=torch.int64, device=DEV)

    def step():
        a, k, c = x.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = rnnt_amd.dense(a, k, c, "gelu", r, 0.2, 5, off)
        return (y, *torch.autograd.grad(y, (a, k, c), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(eager, step()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        x.mul_(0.9)
        off.fill_(2 ** 32 - 1 + i)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, step()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 5000, 300), (2, 1030, 65), (3, 77, 1001), (4, 512, 513), (7, 1024, 64), (8, 2500, 130), (8, 4096, 20000)])
def test_few_rows(M, K, N, dtype):
    """The decoder's form: no gradients, every epilogue."""
    x, w, b, r, _ = data(M, K, N, dtype, 11, residual=True)
    y = rnnt_amd.dense(x.to(DEV), w.to(DEV), b.to(DEV), "silu", r.to(DEV), 0.2, 3, 4)
    X, W = f64(x), f64(w)
    scale = orc.dropout_scale(M, N, 0.2, 3, 4)
    z = X @ W + f64(b)
    want = orc.activation(z, "silu")[0] * scale + f64(r)
    ey = scale * (1.13 * acc(K, np.abs(X) @ np.abs(W) + np.abs(f64(b))) + 2.0 ** -21 * (1 + np.abs(z))) + 2.0 ** -23 * (np.abs(want) + np.abs(f64(r)))
    assert (np.abs(f64(y) - want) <= ey + np.maximum(U[dtype] * (np.abs(want) + ey), LEAST[dtype])).all()


def test_gradient_of_the_gradient_is_refused():
    x, w = torch.ones(4, 8, device=DEV, requires_grad=True), torch.ones(8, 6, device=DEV)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(rnnt_amd.dense(x, w, activation="gelu").sum(), x, create_graph=True)


def test_refusals():
    x, w = torch.zeros(4, 8, device=DEV), torch.zeros(8, 6, device=DEV)
    for args, kw in (((x, w[:7]), {}), ((x, w[0]), {}), ((x, w, w[0, :5]), {}), ((x, w), {"residual": x}), ((x, w), {"activation": "elu"}),
                     ((x, w), {"dropout": 1.0}), ((x, w), {"dropout": 0.5, "seed": -1}), ((x, w[:, :0]), {}), ((x, w.cpu()), {})):
        with pytest.raises(ValueError):
            rnnt_amd.dense(*args, **kw)
    for args, kw in (((x.double(), w.double()), {}), ((x, w.half()), {}), ((x, w), {"residual": torch.zeros(4, 6, device=DEV).bfloat16()}),
                     ((x, w, torch.zeros(6, device=DEV).half()), {})):
        with pytest.raises(TypeError):
            rnnt_amd.dense(*args, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["tanh", "gelu", "silu"])
@pytest.mark.parametrize("rows", [8, 400])
def test_activations_of_small_numbers_are_relative(dtype, act, rows):
    """With one input and a kernel of ones z is x itself, and the result's error is relative to it: 2^-20 for tanh's formula; Phi
    and the logistic function are 1/2 + O(z), off by 1.5e-6 < 2^-18 of that at most; half a step for the type."""
    z = torch.logspace(-36 if dtype != torch.float16 else -7, 0, rows, dtype=torch.float64).to(dtype)
    z[1::2] *= -1
    y = rnnt_amd.dense(z.to(DEV)[:, None], torch.ones(1, 9, dtype=dtype, device=DEV), None, act)
    want = orc.activation(f64(z), act)[0][:, None]
    tol = (2.0 ** -18 + U[dtype] * 1.01) * np.abs(want) + 2 * LEAST[dtype] + 2.0 ** -125
    assert (np.abs(f64(y) - want) <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(33, 2048, 2000), (64, 8, 2048), (50, 1992, 4104), (64, 2048, 8192), (64, 2056, 8192)])
def test_some_rows_of_a_wide_layer(M, K, N, dtype):
    check_layer(M, K, N, dtype, "silu", True, True, 0.2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [8, 600])
def test_gelu_keeps_its_digits_in_the_negative_tail(dtype, rows):
    """z Phi(z) between -12.5 and -1, relative to itself.  With a kernel of one, z is x: exact in 16 bits; the three parts of a float32
    are each summed once, 4 x 2^-24 of z at most, which the tail, exp(-z^2/2), takes z^2 times.
    float32: e^(-z^2/2) has an argument off by 2.5 x 2^-24 of itself: 1.25 z^2 2^-24; the fit 2 x 2^-24, reciprocal, polynomial, exp2 and
    the products 20 roundings or less.  16 bits: 2^-13 by the fit where float16 results are not zero, 2^-9.8 further out; half a step of
    the type."""
    z = torch.linspace(-12.5, -1.0, rows, dtype=torch.float64).to(dtype)
    x = z.to(DEV)[:, None].requires_grad_(True)
    y = rnnt_amd.dense(x, torch.ones(1, 5, dtype=dtype, device=DEV), None, "gelu")
    f = f64(z)
    phi = np.array([0.5 * math.erfc(-v / math.sqrt(2.0)) for v in f])
    want = (f * phi)[:, None]
    rel = (5.25 * f * f + 24) * 2.0 ** -24 if dtype == torch.float32 else np.where(f > -5.9, 2.0 ** -13, 2.0 ** -9.8) + U[dtype] * 1.01
    assert (np.abs(f64(y) - want) <= rel[:, None] * np.abs(want) + LEAST[dtype]).all()
    if dtype == torch.bfloat16:
        return  # its slope comes from a float16 pre-activation
    # Phi(z) + z phi(z): from z = -1.2 on the two terms' sizes add up to 3 times their sum's at most; dz is rounded to the type, the gradient
    # is one column of it times a kernel of one, rounded again
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y) * torch.tensor([1.0, 0, 0, 0, 0], dtype=dtype, device=DEV))
    slope = phi + f * np.exp(-f * f / 2) / math.sqrt(2 * math.pi)
    rel = (5.25 * f * f + 24) * 3 * 2.0 ** -24 + (0 if dtype == torch.float32 else U[dtype] * 2.02)
    far = f <= -1.2
    assert (np.abs(f64(dx)[:, 0] - slope) <= rel * np.abs(slope) + 2 * LEAST[dtype])[far].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,N,act,rate", [(3500, 3400, 136, "silu", 0.1), (9000, 2000, 2100, "gelu", 0.0), (3333, 3531, 205, "linear", 0.0)])
def test_gradients_in_the_largest_blocks(M, K, N, act, rate, dtype):
    """Blocks of 256 x 256 begin at 192 of them: for dx 14 x 14 over rows and inputs (3500 x 3400; 3333 x 3531 with every operand
    packed), for the kernel 8 x 9 over inputs and outputs (2000 x 2100) times 3 pieces of 4096 of the 9000 rows, tiles cut along them and joined."""
    check_layer(M, K, N, dtype, act, True, False, rate)
