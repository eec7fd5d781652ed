"""The beam step against the float64 oracle.  Places (parents, tokens) have to be equal; a total is a float64 sum rounded to
float32, whose log sum exp comes from float32 exponentials good to 2 units in the last place (2^-22 relative, so 2^-22 absolute in the
logarithm): tolerance 2^-24 |total| + 2^-22."""
import numpy as np
import pytest
import torch

import rnnt_amd
from oracle import operators as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def compare(got, want):
    s, p, t = (x.cpu().numpy() for x in got)
    np.testing.assert_array_equal(p, want[1])
    np.testing.assert_array_equal(t, want[2])
    there = want[1] >= 0
    assert (s[~there] == -np.inf).all()
    assert (np.abs(s[there] - want[0][there]) <= 2.0 ** -24 * 1.01 * np.abs(want[0][there]) + 2.0 ** -22).all()


def case(B, K, V, dtype, seed, enc=False, allowed=None, finished=False, scale=3.0):
    rng = np.random.default_rng(seed)
    def t(*shape, s=scale):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * s).to(dtype)
    kw = {}
    if enc:
        kw["enc"] = t(B, V)
    if allowed:
        kw["allowed"] = torch.from_numpy(rng.random((V,) if allowed == "one" else (B, V)) < 0.6)
    if finished:
        kw["finished"] = torch.from_numpy(rng.random((B, K)) < 0.3)
        kw["end"] = int(rng.integers(V))
    scores = torch.from_numpy((-rng.random((B, K)) * 6 - 10).astype(np.float32))
    return t(B, K, V), scores, kw


def run(logits, scores, width, kw):
    got = rnnt_amd.beam_select(logits.to(DEV), scores.to(DEV), width, **{k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()})
    want = orc.beam_select(logits.float().numpy(), scores.numpy(), width, **{k: (v.float() if v.is_floating_point() else v).numpy() if torch.is_tensor(v) else v
                                                                            for k, v in kw.items()})
    compare(got, want)
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,K,V,W", [(1, 1, 1, 1), (1, 4, 62, 4), (2, 3, 7, 8), (3, 5, 512, 9), (2, 8, 513, 16), (1, 17, 1024, 20), (2, 2, 1025, 64), (2, 64, 40, 64),
                                     (1, 16, 2048, 33), (2, 4, 2049, 4), (1, 3, 4100, 17), (2, 9, 10007, 32), (1, 1, 40000, 64), (1, 64, 2100, 64)])
def test_sizes(B, K, V, W, dtype):
    run(*case(B, K, V, dtype, B * 1000 + V)[:2], W, {})


@pytest.mark.parametrize("V", [50, 1000, 3001])
@pytest.mark.parametrize("opts", [{"enc": True}, {"allowed": "one"}, {"allowed": "each"}, {"finished": True}, {"enc": True, "allowed": "each", "finished": True}])
def test_options(V, opts):
    for dtype in (torch.float32, torch.bfloat16):
        logits, scores, kw = case(3, 6, V, dtype, V, **opts)
        run(logits, scores, 6, kw)


@pytest.mark.parametrize("V", [100, 5000])
def test_ties_go_to_the_lowest_place(V):
    logits = torch.zeros(2, 3, V)
    scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -2.0]])
    run(logits, scores, 40, {})
    run(logits.bfloat16(), scores, 64, {"allowed": torch.arange(V) % 3 == 1})
    few = (torch.arange(V) % 5).float().expand(2, 3, V).contiguous()  # every value many times, ascending within a lane
    run(few, scores, 33, {})
    zero = torch.zeros(1, 1, V)
    zero[0, 0, 1::2] = -0.0  # the two zeros are one value
    run(zero, torch.zeros(1, 1), 17, {})


@pytest.mark.parametrize("V", [300, 6000])
def test_adverse_orders(V):
    # everything worth keeping in one lane's values, in one piece, in one beam
    up = torch.arange(V).float() * 1e-3
    scores = torch.zeros(1, 4)
    logits = torch.stack([up, up.flip(0), torch.zeros(V), up * 2]).unsqueeze(0)
    run(logits, scores, 64, {})
    lane = torch.zeros(1, 2, V)
    lane[0, 1, (torch.arange(V) // 8) % 64 == 5] = 4 + torch.rand(int(((torch.arange(V) // 8) % 64 == 5).sum()), generator=torch.Generator().manual_seed(1))
    run(lane, torch.zeros(1, 2), 50, {})


@pytest.mark.parametrize("V", [64, 2500])
def test_empty_beams_and_masked_junk(V):
    logits, _, _ = case(4, 4, V, torch.float32, 3)
    inf, nan = float("inf"), float("nan")
    scores = torch.tensor([[0.0, -inf, -inf, -inf], [-inf] * 4, [nan, -1.0, -3e38, 2e9], [-1e9, -1e9, -5.0, -1e9]])
    run(logits, scores, 8, {})
    ok = torch.arange(V) < V - 9
    for junk in (inf, -inf, nan, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min):
        dirty = logits.clone()
        dirty[:, :, ~ok] = junk
        run(dirty, scores, 8, {"allowed": ok})
    run(logits, scores, 4, {"allowed": torch.zeros(V, dtype=torch.bool)})  # nothing is left anywhere
    one = torch.zeros(4, V, dtype=torch.bool)
    one[0, 3] = one[2, V - 1] = True
    run(logits, torch.zeros(4, 4), 6, {"allowed": one})


@pytest.mark.parametrize("V", [70, 4500])
def test_rows_without_a_probability(V):
    inf, nan = float("inf"), float("nan")
    logits, scores, _ = case(2, 5, V, torch.float32, 5)
    logits[0, 0, 3] = nan
    logits[0, 1, V - 1] = inf
    logits[0, 2] = -inf
    logits[0, 3, 1:] = -inf
    logits[1, 0] = torch.finfo(torch.float32).min  # a mask of the lowest value, over a whole row: uniform
    logits[1, 1, 5:] = torch.finfo(torch.float32).min
    logits[1, 2, :V // 2] = -1e30
    run(logits, scores, 6, {})
    run(logits, torch.tensor([[0.0] * 5, [-inf, -7.0, -inf, -inf, -inf]]), 12, {})
    few = torch.full((1, 2, V), -inf)
    few[0, 0, 7] = few[0, 1, 60] = few[0, 1, 8] = 1.0
    run(few, torch.zeros(1, 2), 9, {})


def test_finished_beams_and_their_scores():
    V = 20
    logits, scores, _ = case(2, 3, V, torch.float32, 6)
    logits[0, 1] = float("nan")  # a finished beam's logits are not looked at
    fin = torch.tensor([[False, True, False], [True, True, True]])
    scores[1] = torch.tensor([-0.0, 0.0, -1.0])
    run(logits, scores, 5, {"finished": fin, "end": V - 1})
    got = run(logits, torch.tensor([[-1.0, float("nan"), -1.0], [float("-inf"), -3.0, -2.0]]), 4, {"finished": fin, "end": 0})
    assert got[1][1].tolist() == [2, 1, -1, -1]


def test_strides():
    big = torch.randn(6, 10, 900, generator=torch.Generator().manual_seed(7)).to(DEV)
    for view in (big[::2, 1:5, 3:703], big.transpose(0, 1), big[:, :, ::3], big[:1].expand(3, 10, 900), big[:, :1].expand(6, 4, 900)):
        B, K, V = view.shape
        scores = -torch.rand(K, B, device=DEV).t()
        a = rnnt_amd.beam_select(view, scores, 5)
        b = rnnt_amd.beam_select(view.contiguous(), scores.contiguous(), 5)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    m = torch.rand(900, 6, device=DEV) < 0.5
    e = torch.randn(900, 6, device=DEV)
    a = rnnt_amd.beam_select(big, torch.zeros(6, 10, device=DEV), 7, enc=e.t(), allowed=m.t())
    b = rnnt_amd.beam_select(big, torch.zeros(6, 10, device=DEV), 7, enc=e.t().contiguous(), allowed=m.t().contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_agrees_with_joint_log_softmax():
    rng = np.random.default_rng(8)
    enc = torch.from_numpy(rng.standard_normal((3, 62)).astype(np.float32)).to(DEV)
    pred = torch.from_numpy(rng.standard_normal((3, 4, 62)).astype(np.float32)).to(DEV)
    scores = -torch.rand(3, 4, device=DEV) * 3
    s, p, t = rnnt_amd.beam_select(pred, scores, 4, enc=enc)
    logp = rnnt_amd.joint_log_softmax(enc, pred.reshape(12, 62), torch.arange(3).repeat_interleave(4), torch.arange(12)).reshape(3, 4, 62)
    want, flat = (scores.unsqueeze(2) + logp).reshape(3, -1).topk(4)
    assert torch.equal(p.long() * 62 + t, flat)
    torch.testing.assert_close(s, want, atol=1e-5, rtol=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int64, torch.bool, torch.uint8, torch.float64])
@pytest.mark.parametrize("tail", [(), (1,), (5,), (250,), (3, 7), (4099,)])
def test_reorder(dtype, tail):
    g = torch.Generator().manual_seed(9)
    B, K, W = 3, 4, 6
    parent = torch.randint(-1, K, (B, W), generator=g, dtype=torch.int32)
    parent[0, 0], parent[2, 5] = K, -7  # outside: zeros
    base = [torch.randint(0, 2 if dtype == torch.bool else 100, (2, B, K) + tail, generator=g).to(dtype) for _ in range(3)]
    out = rnnt_amd.beam_reorder(parent.to(DEV), [s.to(DEV) for s in base], batch_dim=1)
    flat = rnnt_amd.beam_reorder(parent.to(DEV), [s[0].to(DEV) for s in base])
    ok = (parent >= 0) & (parent < K)
    for s, o, f in zip(base, out, flat):
        want = s[:, torch.arange(B)[:, None], parent.clamp(0, K - 1).long()]
        want = torch.where(ok.reshape((1, B, W) + (1,) * len(tail)), want, torch.zeros_like(want))
        assert torch.equal(o.cpu(), want) and torch.equal(f.cpu(), want[0])


def test_reorder_many_tensors_layouts_and_out():
    g = torch.Generator().manual_seed(10)
    B, K, W = 2, 3, 2
    parent = torch.tensor([[2, 0], [-1, 1]], dtype=torch.int32, device=DEV)
    states = [torch.randn(B, K, 5 + i, generator=g).to(DEV) for i in range(35)]  # more than one launch takes
    states[3] = torch.randn(7, K, B, generator=g).to(DEV).permute(2, 1, 0)  # rows that are not dense
    states[4] = torch.randn(B, 1, 9, generator=g).to(DEV).expand(B, K, 9)
    states[5] = torch.randn(B, 6, 9, generator=g).to(DEV)[:, ::2]
    states[6] = torch.zeros(B, K, 0, device=DEV)
    def want(s):
        w = s[torch.arange(B, device=DEV)[:, None], parent.clamp(min=0).long()]
        w[1, 0] = 0
        return w
    for s, o in zip(states, rnnt_amd.beam_reorder(parent, states)):
        assert torch.equal(o, want(s))
    outs = [torch.full((B, W) + s.shape[2:], 9.0, device=DEV) for s in states]
    kept = rnnt_amd.beam_reorder(parent, states, out=outs)
    assert all(a is b and torch.equal(a, want(s)) for a, b, s in zip(kept, outs, states))
    deep = torch.randn(2, 3, B, K, 4, generator=g).to(DEV)
    assert torch.equal(rnnt_amd.beam_reorder(parent, [deep], batch_dim=2)[0], torch.stack([torch.stack([want(y) for y in x]) for x in deep]))
    part = torch.randn(6, B, K, 4, generator=g).to(DEV)[::2, :, :, 1:3]
    assert torch.equal(rnnt_amd.beam_reorder(parent, [part], batch_dim=1)[0], torch.stack([want(x) for x in part]))
    assert rnnt_amd.beam_reorder(parent, []) == []


def test_refusals():
    z = torch.zeros(2, 3, 8, device=DEV)
    s = torch.zeros(2, 3, device=DEV)
    for args, kw in (((z[0], s, 2), {}), ((z, s[:1], 2), {}), ((z, s.double(), 2), {}), ((z, s, 0), {}), ((z, s, 65), {}),
                     ((z, s, 2), {"enc": z[0]}), ((z, s, 2), {"enc": z[:, 0].half()}), ((z, s, 2), {"allowed": z[0, 0]}),
                     ((z, s, 2), {"allowed": torch.ones(3, 8, dtype=torch.bool, device=DEV)}), ((z, s, 2), {"finished": s}),
                     ((z, s, 2), {"finished": s > 0, "end": 8}), ((torch.zeros(1, 65, 4, device=DEV), torch.zeros(1, 65, device=DEV), 2), {}),
                     ((z[:, :, :0], s, 2), {}), ((z, s.cpu(), 2), {})):
        with pytest.raises(ValueError):
            rnnt_amd.beam_select(*args, **kw)
    with pytest.raises(TypeError):
        rnnt_amd.beam_select(z.double(), s, 2)
    p = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    for args, kw in (((p.long(), [z]), {}), ((p[0], [z]), {}), ((p, [z[:1]]), {}), ((p, [z, z[:, :2]]), {}), ((p, [z]), {"batch_dim": 2}), ((p, [z]), {"batch_dim": -1}),
                     ((p, [z]), {"out": [z[:, :2].contiguous().half()]}), ((p, [z]), {"out": []}), ((p, [z[:, :2]]), {"out": [z.view(-1)[:32].view(2, 2, 8)]}),
                     ((p, [z, z]), {"out": [z.new_zeros(2, 2, 8)] * 2})):
        with pytest.raises(ValueError):
            rnnt_amd.beam_reorder(*args, **kw)


def test_step_on_another_stream_and_in_a_graph():
    """Selection and reordering as a decoder runs them, captured once and replayed over three steps."""
    for V in (62, 3000):
        logits = torch.randn(2, 4, V, generator=torch.Generator().manual_seed(11)).to(DEV)
        scores = torch.zeros(2, 4, device=DEV)
        scores[:, 1:] = float("-inf")
        h = torch.randn(3, 2, 4, 16, generator=torch.Generator().manual_seed(12)).to(DEV)

        def step():
            s, p, t = rnnt_amd.beam_select(logits, scores, 4)
            return s, p, t, rnnt_amd.beam_reorder(p, [h], batch_dim=1)[0]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for i in range(3):
            logits.mul_(0.7).add_(0.01 * i)
            scores.copy_(out[0] if i else scores)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_reorder_of_conjugate_and_negated_views():
    """Views whose memory does not hold the values they stand for."""
    s = torch.randn(2, 3, 5, dtype=torch.complex64, device=DEV)
    parent = torch.tensor([[2, 0], [1, 1]], dtype=torch.int32, device=DEV)
    index = parent.long()[..., None].expand(2, 2, 5)
    for v in (s.conj(), s.conj().imag):
        (got,) = rnnt_amd.beam_reorder(parent, [v])
        assert torch.equal(got, v.resolve_conj().resolve_neg().gather(1, index))


@pytest.mark.parametrize("W", [7, 32, 64])
@pytest.mark.parametrize("spread", [0.5, 40.0])
def test_lists_of_many_pieces(W, spread):
    """What the second launch chooses from: beams alike, in order, and one that has everything; equal values everywhere; more lists than
    a block has lanes; 64 pieces a row and one more; finished and empty beams among them."""
    for B, K, V, dtype in ((1, 32, 12000, torch.float16), (1, 64, 33000, torch.bfloat16), (1, 3, 131072, torch.float32), (1, 3, 131073, torch.bfloat16)):
        logits, scores, kw = case(B, K, V, dtype, K + V, finished=K == 3)
        scores = scores - spread * torch.arange(K)
        scores[0, K // 2] = float("nan")
        run(logits, scores, W, kw)
        if K == 32:
            run(logits[:, :1].expand(B, K, V).contiguous(), torch.full((B, K), -1.0), W, kw)
    run(torch.zeros(2, 20, 6000), -spread * torch.arange(40).reshape(2, 20).float(), W, {})


def test_reorder_of_a_state_with_a_dimension_of_size_one():
    """[layers, 1, B, K, hidden] made by transposing [1, layers, ...]: dense, though the stride of its dimension of size 1 is not the
    distance of the layers."""
    base = torch.randn(1, 3, 2, 4, 5, generator=torch.Generator().manual_seed(13)).to(DEV)
    s = base.transpose(0, 1)
    assert s.is_contiguous() and s.stride(1) != s.stride(0)
    parent = torch.tensor([[2, 0, 3], [-1, 1, 1]], dtype=torch.int32, device=DEV)
    (got,) = rnnt_amd.beam_reorder(parent, [s], batch_dim=2)
    want = s[:, :, torch.arange(2, device=DEV)[:, None], parent.clamp(min=0).long()]
    want[:, :, 1, 0] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("V", [2048, 1024, 6 * 2048])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_flat_tails(V, dtype):
    """One peak over 1023 or 2047 symbols of one value, whose terms are all off by the same amount: nothing averages out.  The sum's error
    is that of a term, 2^-24 (1.43 + ln 2) for exp2 and its argument, below 2^-22, on top of half a step of the total."""
    g = torch.Generator().manual_seed(14)
    n = 60
    tail = torch.randn(n, generator=g) * 10.0 ** (torch.rand(n, generator=g) * 6 - 5)
    peak = tail + 5 + 11 * torch.rand(n, generator=g)
    logits = tail.to(dtype)[:, None].expand(n, V).clone()
    logits[:, 77::2048] = peak.to(dtype)[:, None]  # long rows are summed in pieces of 2048: a peak in each
    run(logits.reshape(4, 15, V), -torch.rand(4, 15, generator=g) * 1e-3, 15, {})


@pytest.mark.parametrize("pieces", [1, 3])
def test_beams_whose_totals_are_nearly_the_same(pieces):
    """Two beams whose best totals are 5e-7 apart, over flat tails of different depth.  The logarithm of a row's sum is good to
    2.12 x 2^-24 (a term's error), twice that is 2.6e-7."""
    rows = [(5.9910145, 0.27237773), (5.874392, 0.15194488)]
    V = 2048 * pieces
    logits = torch.empty(1, 2, V)
    for k, (peak, tail) in enumerate(rows):
        logits[0, k] = tail
        logits[0, k, 5::2048] = peak
    x = logits.double()
    lse = torch.logsumexp(x - x.amax(2, keepdim=True), 2)[0]
    for gap in (5e-7, -5e-7):
        run(logits, torch.tensor([[(lse[0] - lse[1] + gap).item(), 0.0]]), 2, {})


def test_reorder_into_out_is_seen_by_autograd():
    """`out` is written in place: a graph that keeps it raises instead of using what is there now, and a tensor that requires
    gradients is refused as any in-place write of one is."""
    parent = torch.tensor([[2, 0], [1, 1]], dtype=torch.int32, device=DEV)
    state, out = torch.randn(2, 3, 5, device=DEV), torch.randn(2, 2, 5, device=DEV)
    w = torch.ones(5, device=DEV, requires_grad=True)
    y = (out[0] * w).sum()  # a view keeps it, too
    before = out._version
    rnnt_amd.beam_reorder(parent, [state], out=[out])
    assert out._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    leaf = torch.zeros(2, 2, 5, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="require gradients"):
        rnnt_amd.beam_reorder(parent, [state], out=[leaf])
    with torch.no_grad():
        assert torch.equal(rnnt_amd.beam_reorder(parent, [state], out=[leaf])[0], rnnt_amd.beam_reorder(parent, [state])[0])
    with torch.inference_mode():
        fixed = torch.zeros(2, 2, 5, device=DEV)
        rnnt_amd.beam_reorder(parent, [state], out=[fixed])
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        rnnt_amd.beam_reorder(parent, [state], out=[fixed])
