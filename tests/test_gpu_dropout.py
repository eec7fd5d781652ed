"""Dropout with a mask that is never stored, against the float64 oracle.  y = x * c with c = 1/keep in float32: the scale and
the product are each rounded to float32, and 16-bit types round once more; a tolerance counts half a step for each."""
import numpy as np
import pytest
import torch

import rnnt_amd
from oracle import operators as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def tol(dtype):
    return 2 * 2.0 ** -24 * 1.01 + (0 if dtype == torch.float32 else HALF[dtype] * 1.01)


def make(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def check(y, x, rate, seed, offset):
    want = x.double().numpy().reshape(-1, x.shape[-1]) * orc.dropout_scale(x.numel() // x.shape[-1], x.shape[-1], rate, seed, offset)
    got = y.detach().double().cpu().numpy().reshape(want.shape)
    assert ((got == 0) == (want == 0)).all()
    # float16 values below 2^-14 lie 2^-24 apart whatever their size, so their rounding is off by up to 2^-25
    least = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    assert (np.abs(got - want) <= np.maximum(tol(x.dtype) * np.abs(want), least)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 8), (3, 1), (5, 7), (33, 62), (129, 250), (2, 3, 64), (1100, 9), (3, 4097), (2, 70001)])
def test_forward_and_backward(shape, dtype):
    x = make(shape, dtype, 1)
    x[x == 0] = 1
    xd = x.to(DEV).requires_grad_(True)
    y = rnnt_amd.dropout(xd, 0.3, seed=2 ** 50 + 3, offset=2 ** 40 + 11)
    check(y, x, 0.3, 2 ** 50 + 3, 2 ** 40 + 11)
    dy = make(shape, dtype, 2)
    dy[dy == 0] = 1
    (dx,) = torch.autograd.grad(y, xd, dy.to(DEV))
    check(dx, dy, 0.3, 2 ** 50 + 3, 2 ** 40 + 11)


def test_very_long_row_takes_the_division_of_long_rows():
    x = torch.ones(2, 600_001)
    y = rnnt_amd.dropout(x.to(DEV), 0.5, seed=1, offset=0)
    check(y, x, 0.5, 1, 0)


def test_strides_and_other_layouts():
    base = make((40, 70), torch.float32, 3).to(DEV)
    for view in (base[:, :33], base.t(), base[::2], base[3:, 5:64], base.reshape(4, 10, 70)[:, 1:3, ::2]):
        assert torch.equal(rnnt_amd.dropout(view, 0.4, seed=4), rnnt_amd.dropout(view.contiguous(), 0.4, seed=4))
    scalar = torch.tensor(2.0, device=DEV)
    assert rnnt_amd.dropout(scalar, 0.5, seed=1).shape == ()


def test_rates():
    x = make((64, 100), torch.float32, 5).to(DEV)
    assert rnnt_amd.dropout(x, 0.0) is x
    assert rnnt_amd.dropout(x[:0], 0.5).shape == (0, 100)
    check(rnnt_amd.dropout(x, 65535 / 65536, seed=9), x.cpu(), 65535 / 65536, 9, 0)
    check(rnnt_amd.dropout(x, 2 ** -16, seed=9), x.cpu(), 2 ** -16, 9, 0)


def test_dropped_infinities_and_nans_are_zero_and_kept_ones_stay():
    x = torch.full((16, 64), float("inf"))
    x[::2] = float("nan")
    kept = orc.dropout_scale(16, 64, 0.5, 7, 0) > 0
    y = rnnt_amd.dropout(x.to(DEV), 0.5, seed=7).cpu().numpy()
    assert (y[~kept] == 0).all() and not np.isfinite(y[kept]).any()


def test_seeds_and_offsets_give_other_masks():
    x = torch.ones(256, 256, device=DEV)
    a = rnnt_amd.dropout(x, 0.5, seed=1, offset=0)
    assert torch.equal(a, rnnt_amd.dropout(x, 0.5, seed=1, offset=0))
    for kw in ({"seed": 2}, {"seed": 1 + 2 ** 32}, {"seed": 1, "offset": 1}, {"seed": 1, "offset": 2 ** 32}):
        same = (a == rnnt_amd.dropout(x, 0.5, **kw)).float().mean().item()
        assert abs(same - 0.5) < 5 * 0.5 / 256


def test_offset_in_device_memory_and_graph_replays():
    x = make((50, 130), torch.bfloat16, 6).to(DEV)
    off = torch.tensor([2 ** 33 + 5], device=DEV)
    assert torch.equal(rnnt_amd.dropout(x, 0.25, seed=3, offset=off), rnnt_amd.dropout(x, 0.25, seed=3, offset=2 ** 33 + 5))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rnnt_amd.dropout(x, 0.25, seed=3, offset=off)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rnnt_amd.dropout(x, 0.25, seed=3, offset=off)
        off.add_(1)
    for i in range(4):
        off.fill_(100 + i)
        g.replay()
        assert torch.equal(y, rnnt_amd.dropout(x, 0.25, seed=3, offset=100 + i))
        assert off.item() == 101 + i


def test_backward_refuses_an_offset_that_has_moved():
    x = torch.ones(4, 8, device=DEV, requires_grad=True)
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    y = rnnt_amd.dropout(x, 0.5, seed=1, offset=off)
    off.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradient_of_the_gradient():
    x = torch.randn(5, 9, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad((rnnt_amd.dropout(x, 0.5, seed=3) ** 2).sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(g.sum(), x)
    scale = torch.from_numpy(orc.dropout_scale(5, 9, 0.5, 3, 0)).to(DEV)
    assert torch.equal(gg.double(), 2 * scale ** 2)


def test_refusals():
    x = torch.zeros(3, 4, device=DEV)
    with pytest.raises(TypeError):
        rnnt_amd.dropout(x.double(), 0.1)
    with pytest.raises(TypeError):
        rnnt_amd.dropout(x.int(), 0.1)
    for rate in (-0.5, 1.0, float("nan")):
        with pytest.raises(ValueError):
            rnnt_amd.dropout(x, rate)
    with pytest.raises(ValueError):
        rnnt_amd.dropout(x, 0.1, offset=torch.zeros(1, dtype=torch.int64))
