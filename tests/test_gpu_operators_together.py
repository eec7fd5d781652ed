"""The operators as they are used together: a training step of the fully-connected joint with dropout against float64, and a
decoder's steps (dense on the beam's rows, selection, states in their new order) against the float64 oracle."""
import gc

import numpy as np
import pytest
import torch

import rnnt_amd
from oracle import operators as ops
from oracle import rnnt_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _joint(seed, B, T, U, He, Hd, widths, V):
    g = torch.Generator().manual_seed(seed)
    def t(*s, scale=1.0):
        return torch.randn(s, generator=g) * scale
    yt, yp = t(B, T, He), t(B, U + 1, Hd)
    sizes = [He + Hd, *widths, V]
    weights = [(t(a, b, scale=a ** -0.5), t(b, scale=0.1)) for a, b in zip(sizes, sizes[1:])]
    lab = torch.randint(0, V - 1, (B, U), generator=g, dtype=torch.int32)
    return yt, yp, weights, lab


@pytest.mark.parametrize("widths", [(24,), (40, 30), (150, 33, 20)])
def test_training_step_of_the_joint_with_dropout(widths):
    B, T, U, He, Hd, V, rate, seed, offset = 2, 9, 4, 20, 12, 17, 0.3, 5, 2 ** 40
    yt, yp, weights, lab = _joint(1, B, T, U, He, Hd, widths, V)
    il, ll = torch.tensor([[9], [7]], dtype=torch.int32), torch.tensor([[4], [2]], dtype=torch.int32)
    dev = [t.to(DEV).requires_grad_(True) for t in (yt, yp, *[w for p in weights for w in p])]
    pairs = list(zip(dev[2::2], dev[3::2]))
    costs = rnnt_amd.fc_joint_loss(dev[0], dev[1], pairs, lab.to(DEV), il.to(DEV), ll.to(DEV), blank_label=V - 1, dropout=rate, seed=seed, offset=offset)
    grads = torch.autograd.grad(costs.mean(), dev)

    # float64 on the host: the joint by autograd with the masks as constants, the loss and its gradient by the oracle
    ref = [t.double().requires_grad_(True) for t in (yt, yp, *[w for p in weights for w in p])]
    h = torch.cat([ref[0][:, 2:].unsqueeze(2).expand(-1, -1, U + 1, -1), ref[1].unsqueeze(1).expand(-1, T - 2, -1, -1)], dim=-1)
    for i, (k, b) in enumerate(zip(ref[2::2], ref[3::2])):
        h = h @ k + b
        if i < len(weights) - 1:
            h = torch.tanh(h)
            m = ops.dropout_scale(B * (T - 2) * (U + 1), h.shape[-1], rate, seed, offset + i)
            h = h * torch.from_numpy(m).reshape(h.shape)
    want, d_acts = orc.rnnt_loss_and_grad(h.detach().numpy(), lab.numpy(), (il - 2).reshape(B).numpy(), ll.reshape(B).numpy(), V - 1, np.full(B, 1.0 / B))
    np.testing.assert_allclose(costs.detach().cpu().numpy(), want, rtol=1e-5)
    for g, r in zip(grads, torch.autograd.grad(h, ref, torch.from_numpy(np.asarray(d_acts, np.float64)))):
        # the loss's own bar on d_acts is 1e-4 absolute (2e-5 measured); a gradient of a weight sums up to B T (U+1) of them
        assert (g.cpu().double() - r).abs().max() < 1e-4 * max(1.0, r.abs().max().item())


def test_no_dropout_is_what_it_was():
    yt, yp, weights, _ = _joint(2, 2, 6, 3, 10, 8, (20, 12), 9)
    args = yt.to(DEV), yp.to(DEV), [(k.to(DEV), b.to(DEV)) for k, b in weights]
    assert torch.equal(rnnt_amd.fc_joint(*args), rnnt_amd.fc_joint(*args, dropout=0.0, seed=3, offset=9))
    with pytest.raises(ValueError):
        rnnt_amd.fc_joint(*args, dropout=1.0)


def test_an_offset_in_device_memory_gives_the_same_step():
    yt, yp, weights, _ = _joint(3, 1, 5, 2, 6, 6, (16, 16, 8), 7)
    args = yt.to(DEV), yp.to(DEV), [(k.to(DEV), b.to(DEV)) for k, b in weights]
    a = rnnt_amd.fc_joint(*args, dropout=0.5, seed=3, offset=70)
    assert torch.equal(a, rnnt_amd.fc_joint(*args, dropout=0.5, seed=3, offset=torch.tensor([70], device=DEV)))
    assert not torch.equal(a, rnnt_amd.fc_joint(*args, dropout=0.5, seed=3, offset=71))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [62, 2500])
def test_decoder_steps(V, dtype):
    """Three steps of a beam search over a small recurrent prediction network: hidden layer with a skip connection, output layer,
    selection, reordering.  The oracle selects from the very logits the layers gave, in float64."""
    g = torch.Generator().manual_seed(4)
    B, K, H = 3, 4, 48
    def t(*s, scale=1.0):
        return (torch.randn(s, generator=g) * scale).to(dtype).to(DEV)
    w1, b1, w2, b2, emb, enc = t(H, H, scale=H ** -0.5), t(H, scale=0.1), t(H, V, scale=2 * H ** -0.5), t(V, scale=0.1), t(V, H), t(B, V)
    h = t(B, 1, H).expand(B, K, H)
    scores = torch.full((B, K), float("-inf"), device=DEV)
    scores[:, 0] = 0
    finished = torch.zeros(B, K, dtype=torch.bool, device=DEV)
    history = torch.zeros(B, K, 3, dtype=torch.int64, device=DEV)
    for step in range(3):
        h = rnnt_amd.dense(h, w1, b1, "tanh", residual=h)
        logits = rnnt_amd.dense(h, w2, b2)
        args = logits, scores, K
        new, parent, token = rnnt_amd.beam_select(*args, enc=enc, finished=finished, end=0)
        want = ops.beam_select(logits.float().cpu().numpy(), scores.cpu().numpy(), K, enc=enc.float().cpu().numpy(), finished=finished.cpu().numpy(), end=0)
        np.testing.assert_array_equal(parent.cpu().numpy(), want[1])
        np.testing.assert_array_equal(token.cpu().numpy(), want[2])
        np.testing.assert_allclose(new.cpu().numpy(), want[0], rtol=2.0 ** -23, atol=2.0 ** -22)
        before = h.cpu(), history.cpu()
        h, history = rnnt_amd.beam_reorder(parent, [h, history])
        at = torch.arange(B)[:, None], parent.cpu().long()
        assert torch.equal(h.cpu(), before[0][at]) and torch.equal(history.cpu(), before[1][at])
        history[:, :, step] = token
        finished = token == 0
        scores = new
        h = h + emb[token.long()]
    assert scores.isfinite().all() and (scores[:, :-1] >= scores[:, 1:]).all()


def test_captured_backward_pass_of_leaves_that_an_eager_graph_holds_is_refused():
    """It would make a stream outside the capture wait for it; with the eager graph gone the same leaves are captured."""
    x = torch.randn(40, 24, device=DEV)
    w, b = (torch.randn(24, 16, device=DEV) * 0.2).requires_grad_(True), torch.zeros(16, device=DEV, requires_grad=True)

    def step(k):
        y = rnnt_amd.dropout(rnnt_amd.dense(x, k, b, "tanh"), 0.25, seed=3)
        return torch.autograd.grad((y * y).sum(), (k, b))
    eager = rnnt_amd.dense(x, w, b, "tanh")  # holds the leaves' nodes on this stream
    with pytest.raises(RuntimeError, match="eager graph on another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(w)
    held = rnnt_amd.dropout(w, 0.5)
    with pytest.raises(RuntimeError, match="eager graph on another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            (rnnt_amd.dropout(w, 0.5) * 2.0).backward(torch.ones_like(w))
    del eager, held
    gc.collect()  # and what the errors held
    want = step(w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(w)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step(w)))
    assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.parametrize("op", ["dense", "dropout"])
def test_captured_backward_pass_is_refused_where_the_leaf_lies_behind_other_nodes(op):
    """The leaf that the eager graph holds comes several nodes behind the operator's own."""
    x = torch.randn(30, 20, device=DEV)
    w = (torch.randn(20, 16, device=DEV) * 0.2).requires_grad_(True)

    def layer(w):
        k = (w * 1.5).tanh().t().contiguous().t()
        return rnnt_amd.dense(x, k, None, "silu") if op == "dense" else rnnt_amd.dropout(k, 0.25, seed=3)

    def step(w):
        y = layer(w)
        return torch.autograd.grad((y * y).sum(), w)
    eager = w.sin()
    with pytest.raises(RuntimeError, match="eager graph on another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(w)
    del eager
    gc.collect()
    (want,) = step(w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        (out,) = step(w)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("i", range(4))
def test_tensors_without_memory_of_their_own_never_reach_a_kernel(i):
    """Transformed, fake and meta tensors have no data pointer: the calls raise."""
    from torch._subclasses import FakeTensorMode
    parent, k, scores = torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.ones(8, 6, device=DEV), torch.zeros(2, 3, device=DEV)
    call = (lambda x: rnnt_amd.dense(x, k), lambda x: rnnt_amd.dropout(x, 0.5), lambda x: rnnt_amd.beam_select(x, scores, 2)[0],
            lambda x: rnnt_amd.beam_reorder(parent, [x])[0])[i]
    x = torch.randn(2, 3, 8, device=DEV)
    call(x)
    for bad in (lambda: torch.vmap(call)(x[None]), lambda: torch.func.grad(lambda t: call(t).sum())(x), lambda: call(x.to("meta"))):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    with FakeTensorMode(), pytest.raises((RuntimeError, ValueError)):
        call(torch.empty(2, 3, 8, device=DEV))
    torch.cuda.synchronize()


def _negated(t):
    """A view whose memory holds -t."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_negated_views_give_their_values(dtype):
    """What memory holds is not the value: dense, dropout and the beam step, each input in turn, forward and backward."""
    g = torch.Generator().manual_seed(15)
    def t(*s):
        return torch.randn(s, generator=g).to(dtype).to(DEV)
    args = {"x": t(70, 24), "kernel": t(24, 16), "bias": t(16), "residual": t(70, 16)}

    def step(args, dy):
        leaves = {n: a.detach().requires_grad_(True) for n, a in args.items()}
        y = rnnt_amd.dense(**leaves, activation="tanh", dropout=0.2, seed=1, offset=off)
        return (y, *torch.autograd.grad(y, list(leaves.values()), dy))
    off, dy = torch.tensor([9], device=DEV), t(70, 16)
    want = step(args, dy)
    for name in args:
        assert all(torch.equal(a, b) for a, b in zip(step({**args, name: _negated(args[name])}, dy), want)), name
    assert all(torch.equal(a, b) for a, b in zip(step(args, _negated(dy)), want))
    plain, off = off, _negated(off)
    assert all(torch.equal(a, b) for a, b in zip(step(args, dy), want))
    # one column of a complex matrix: dense as it lies, and negated
    z = torch.randn(40, 1, dtype=torch.complex64, generator=g).to(DEV).conj().imag
    if dtype == torch.float32:
        assert z.is_neg()
        k, r = t(1, 5), z.clone()
        assert torch.equal(rnnt_amd.dense(z, k), rnnt_amd.dense(z.clone(), k))
        assert torch.equal(rnnt_amd.dense(args["x"][:40], t(24, 1) * 0, residual=z), r)

    x = args["x"].clone().requires_grad_(True)
    y = rnnt_amd.dropout(_negated(x), 0.4, seed=3, offset=off)
    assert torch.equal(y, rnnt_amd.dropout(x, 0.4, seed=3, offset=plain))
    assert torch.equal(torch.autograd.grad(y, x, _negated(args["x"]))[0], rnnt_amd.dropout(args["x"], 0.4, seed=3, offset=plain))

    logits, scores, enc = t(2, 3, 50), -torch.rand(2, 3, device=DEV), t(2, 50)
    want = rnnt_amd.beam_select(logits, scores, 4, enc)
    for i in range(3):
        given = [_negated(a) if i == j else a for j, a in enumerate((logits, scores, enc))]
        assert all(torch.equal(a, b) for a, b in zip(rnnt_amd.beam_select(given[0], given[1], 4, given[2]), want))
    (moved,) = rnnt_amd.beam_reorder(want[1], [logits])
    assert torch.equal(rnnt_amd.beam_reorder(_negated(want[1]), [_negated(logits)])[0], moved)
    with pytest.raises(ValueError, match="out must be dense"):
        rnnt_amd.beam_reorder(want[1], [logits], out=[torch._neg_view(torch.zeros_like(moved))])
