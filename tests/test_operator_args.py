"""Dropout and beam operators without a GPU: known answers of the generator's oracle, refusals of the C entry points before
any launch, refusals of the Python entry points."""
import ctypes

import numpy as np
import pytest
import torch

import rnnt_amd
from oracle import operators as orc
from rnnt_amd import _lib, _operator

ONE = 4096  # an address that is never dereferenced: validation fails first


def test_philox_known_answers():
    # the published vectors of Philox4x32-10: zeros, all ones, digits of pi
    def words(c, k):
        return [int(w) for w in orc.philox4x32(c, k)]
    assert words((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert words((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_dropout_entry_point_refuses():
    f = _lib.lib().rnnt_mi355x_dropout

    def call(x=ONE, xs=8, y=2 * ONE, rows=4, cols=8, dtype=0, drop=100, seed=1, off=1):
        return f(x, xs, y, rows, cols, dtype, drop, seed, off, None, None)
    for bad in ({"x": None}, {"y": None}, {"rows": 0}, {"cols": 0}, {"xs": 7}, {"drop": -1}, {"drop": 65536}, {"dtype": 3}, {"dtype": -1},
                {"x": ONE, "y": ONE, "xs": 9}):
        assert call(**bad) == _lib.INVALID_VALUE, bad
    assert call(rows=1 << 31) == _lib.UNSUPPORTED_SIZE
    assert call(rows=(1 << 31) - 1, cols=1 << 20, xs=1 << 20) == _lib.UNSUPPORTED_SIZE


def test_beam_select_entry_point_refuses():
    L = _lib.lib()
    n = ctypes.c_size_t(0)
    q = L.rnnt_mi355x_beam_select_workspace_bytes
    assert q(2, 4, 2048, 4, ctypes.byref(n)) == 0 and n.value == 0
    assert q(2, 4, 2049, 4, ctypes.byref(n)) == 0 and n.value == 2 * 4 * 2 * (16 + 8 * 8)
    assert q(2, 4, 2049, 33, ctypes.byref(n)) == 0 and n.value == 2 * 4 * 2 * (16 + 64 * 8)
    assert q(2, 4, 2049, 4, None) == _lib.INVALID_VALUE
    for bad in ((0, 4, 8, 4), (1, 0, 8, 4), (1, 4, 0, 4), (1, 4, 8, 0)):
        assert q(*bad, ctypes.byref(n)) == _lib.INVALID_VALUE
    for big in ((1, 65, 8, 4), (1, 4, 8, 65), (1, 64, 1 << 25, 4), (1 << 20, 64, 1 << 20, 4)):
        assert q(*big, ctypes.byref(n)) == _lib.UNSUPPORTED_SIZE

    def call(logits=ONE, sb=32, sk=8, dtype=0, scores=ONE, finished=None, end=0, B=2, K=4, V=8, width=4, o=ONE, ws=None):
        return L.rnnt_mi355x_beam_select(logits, sb, sk, dtype, None, 0, scores, None, 0, finished, end, B, K, V, width, o, o, o, ws, None)
    for bad in ({"logits": None}, {"scores": None}, {"o": None}, {"sb": -1}, {"sk": -8}, {"dtype": 5}, {"finished": ONE, "end": 8},
                {"finished": ONE, "end": -1}, {"V": 3000, "sk": 3000, "ws": None}, {"width": 0}):
        assert call(**bad) == _lib.INVALID_VALUE, bad
    assert call(width=65) == _lib.UNSUPPORTED_SIZE


def test_beam_reorder_entry_point_refuses():
    f = _lib.lib().rnnt_mi355x_beam_reorder

    def call(n=1, parent=ONE, B=2, K=3, W=4, **kw):
        t = _lib.ReorderTensor(**{"src": ONE, "dst": 2 * ONE, "outer": 1, "outer_stride": 0, "batch_stride": 48, "beam_stride": 16, "row_bytes": 16, **kw})
        return f((_lib.ReorderTensor * 17)(*[t] * 17), n, parent, B, K, W, None)
    for bad in ({"n": 0}, {"parent": None}, {"B": 0}, {"K": 0}, {"W": 0}, {"src": None}, {"dst": None}, {"outer": 0}, {"row_bytes": 0},
                {"outer_stride": -1}, {"batch_stride": -1}, {"beam_stride": -1}):
        assert call(**bad) == _lib.INVALID_VALUE, bad
    assert call(n=17) == _lib.UNSUPPORTED_SIZE
    assert call(outer=1 << 31) == _lib.UNSUPPORTED_SIZE
    assert call(row_bytes=1 << 44) == _lib.UNSUPPORTED_SIZE
    assert f(None, 1, ONE, 1, 1, 1, None) == _lib.INVALID_VALUE


def _layer(**kw):
    return _lib.Layer(**{"x": ONE, "kernel": 2 * ONE, "y": 3 * ONE, "x_stride": 8, "kernel_stride": 6, "rows": 4, "n_in": 8, "n_out": 6, **kw})


def test_layer_entry_points_refuse():
    L = _lib.lib()
    f, b, q = L.rnnt_mi355x_layer_forward, L.rnnt_mi355x_layer_backward, L.rnnt_mi355x_layer_workspace_bytes
    for bad in ({"x": None}, {"kernel": None}, {"y": None}, {"rows": 0}, {"n_in": 0}, {"n_out": 0}, {"x_stride": 7}, {"kernel_stride": 5}, {"dtype": 3},
                {"dtype": -1}, {"act": 5}, {"act": -1}, {"drop16": -1}, {"drop16": 65536}, {"residual": ONE, "residual_stride": 5}):
        assert f(_layer(**bad), None, None) == _lib.INVALID_VALUE, bad
    for big in ({"rows": 1 << 31}, {"n_in": (1 << 24) + 1, "x_stride": 1 << 25}, {"n_out": (1 << 24) + 1, "kernel_stride": 1 << 25}):
        assert f(_layer(**big), None, None) == _lib.UNSUPPORTED_SIZE, big
    assert f(None, None, None) == _lib.INVALID_VALUE
    assert f(_layer(n_in=4000, x_stride=4000), None, None) == _lib.INVALID_VALUE  # split along k: needs its workspace

    def back(layer, dy=ONE, stride=6, ws=ONE):
        return b(layer, dy, stride, ONE, ONE, ONE, ws, None)
    assert back(_layer(), dy=None) == back(_layer(), stride=5) == back(_layer(), ws=None) == back(_layer(x=None)) == _lib.INVALID_VALUE
    # without the pre-activation only what y determines is accepted
    for bad in ({"act": 3}, {"act": 4}, {"act": 1, "dtype": 1}, {"act": 1, "residual": ONE, "residual_stride": 6}, {"act": 2, "residual": ONE, "residual_stride": 6},
                {"act": 2, "y": None}):
        assert back(_layer(**bad)) == _lib.INVALID_VALUE, bad
    n, m = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert q(_layer(), ONE, 6, ctypes.byref(n), ctypes.byref(m)) == 0 and n.value == 0 and m.value >= 24
    assert q(_layer(n_in=4000, x_stride=4000), None, 0, ctypes.byref(n), None) == 0 and n.value > 0
    assert q(_layer(), ONE, 5, None, ctypes.byref(m)) == _lib.INVALID_VALUE
    assert q(None, None, 0, ctypes.byref(n), None) == _lib.INVALID_VALUE


def test_layer_structure_has_the_size_of_the_header():
    assert ctypes.sizeof(_lib.Layer) == 6 * 8 + 4 * 8 + 5 * 4 + 4 + 3 * 8
    assert ctypes.sizeof(_lib.ReorderTensor) == 7 * 8


def test_python_refusals_of_host_tensors():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="MI355X"):
        rnnt_amd.dropout(x, 0.1)
    with pytest.raises(ValueError, match="MI355X"):
        rnnt_amd.beam_select(x, torch.zeros(2, 3), 2)
    with pytest.raises(ValueError, match="MI355X"):
        rnnt_amd.beam_reorder(torch.zeros(2, 2, dtype=torch.int32), [x])
    with pytest.raises(ValueError, match="MI355X"):
        rnnt_amd.dense(x, torch.zeros(8, 4))
    with pytest.raises(TypeError):
        rnnt_amd.dropout([1.0], 0.1)


def test_rates_and_seeds():
    assert _operator.drop16("d", 0.0) == 0 and _operator.drop16("d", 0.5) == 32768 and _operator.drop16("d", 1e-7) == 0
    for bad in (-0.1, 1.0, 1.5, float("nan"), 1 - 2.0 ** -18):
        with pytest.raises(ValueError):
            _operator.drop16("d", bad)
    cpu = torch.device("cpu")
    assert _operator.seed_offset("d", 2 ** 64 - 1, 7, cpu) == (2 ** 64 - 1, 7, None)
    for seed, off in ((-1, 0), (2 ** 64, 0), (0, -1), (0, 2 ** 64), (0, torch.zeros(1)), (0, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            _operator.seed_offset("d", seed, off, cpu)
    t = torch.zeros(1, dtype=torch.int64)
    assert _operator.seed_offset("d", 3, t, cpu) == (3, 0, t)


def test_oracle_of_the_mask_keeps_the_right_share():
    s = orc.dropout_scale(400, 501, 0.3, 5, 9)
    n = s.size
    kept = (s > 0).sum()
    assert abs(kept - 0.7 * n) < 5 * np.sqrt(n * 0.21)
    assert np.allclose(s[s > 0], 1 / 0.7, rtol=1e-4)


def test_beam_select_refuses_a_vocabulary_whose_last_piece_passes_the_int():
    q, n = _lib.lib().rnnt_mi355x_beam_select_workspace_bytes, ctypes.c_size_t(0)
    for V in ((1 << 31) - 1, (1 << 31) - 8, (1 << 31) - 2048, (1 << 31) - (1 << 16) + 1):
        assert q(1, 1, V, 4, ctypes.byref(n)) == _lib.UNSUPPORTED_SIZE
    assert q(1, 1, (1 << 31) - (1 << 16), 4, ctypes.byref(n)) == 0


def test_calls_beyond_a_launch_are_refused():
    """Fewer than 2^32 threads go into one launch."""
    L, n = _lib.lib(), ctypes.c_size_t(0)
    q = L.rnnt_mi355x_beam_select_workspace_bytes
    for big in ((1 << 22, 1, 8, 4), (1 << 20, 32, 4097, 4), ((1 << 22) - 1, 1, 40000, 4)):
        assert q(*big, ctypes.byref(n)) == _lib.UNSUPPORTED_SIZE
    assert q((1 << 22) - 1, 64, 2048, 4, ctypes.byref(n)) == 0 and q((1 << 20) - 1, 32, 4096, 4, ctypes.byref(n)) == 0
    q = L.rnnt_mi355x_layer_workspace_bytes
    assert q(_layer(rows=(1 << 30) - 63), None, 0, ctypes.byref(n), None) == _lib.UNSUPPORTED_SIZE
    assert q(_layer(rows=(1 << 30) - 64), None, 0, ctypes.byref(n), None) == 0


def test_strides_of_a_dense_state_come_from_its_sizes():
    """A dimension of size 1 may carry any stride in a tensor that is dense all the same."""
    strides = _lib.native().reorder_strides
    s = torch.empty(1, 3, 2, 5, 4).transpose(0, 1)  # [3, 1, B, K, 4]
    assert s.is_contiguous() and s.stride(1) == 3 * 40
    assert strides(s, 2) == (3, 40, 20, 4)
    assert strides(torch.empty(2, 5, 4).as_strided((1, 2, 5, 4), (7, 20, 4, 1)), 1) == (1, 40, 20, 4)
    assert strides(torch.empty(6, 2, 5, 4)[::2], 1) == (3, 80, 20, 4)
    assert strides(torch.empty(2, 5), 0) == (1, 10, 5, 1)


def _calls(wrap):
    """Each operator with `wrap` around one of its floating inputs at a time."""
    x, k, b, r = torch.randn(4, 8), torch.randn(8, 6), torch.randn(6), torch.randn(4, 6)
    logits, scores, enc = torch.randn(2, 3, 8), torch.zeros(2, 3), torch.randn(2, 8)
    parent = torch.zeros(2, 3, dtype=torch.int32)
    yield lambda: rnnt_amd.dense(wrap(x), k, b, residual=r)
    yield lambda: rnnt_amd.dense(x, wrap(k), b, residual=r)
    yield lambda: rnnt_amd.dense(x, k, wrap(b), residual=r)
    yield lambda: rnnt_amd.dense(x, k, b, residual=wrap(r))
    yield lambda: rnnt_amd.dropout(wrap(x), 0.5)
    yield lambda: rnnt_amd.beam_select(wrap(logits), scores, 2, enc)
    yield lambda: rnnt_amd.beam_select(logits, wrap(scores), 2, enc)
    yield lambda: rnnt_amd.beam_select(logits, scores, 2, wrap(enc))
    yield lambda: rnnt_amd.beam_reorder(parent, [logits, wrap(logits)])
    yield lambda: rnnt_amd.beam_reorder(parent, [logits], out=[wrap(torch.zeros(2, 3, 8))])


def test_forward_mode_differentiation_is_refused():
    """A dual tensor does not say requires_grad; its tangent would be lost without a word."""
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        for call in _calls(lambda t: fwd.make_dual(t, torch.ones_like(t))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def _operators():
    parent = torch.zeros(2, 3, dtype=torch.int32)
    return (lambda x: rnnt_amd.dense(x, torch.ones(8, 6)), lambda x: rnnt_amd.dropout(x, 0.5),
            lambda x: rnnt_amd.beam_select(x, torch.zeros(2, 3), 2), lambda x: rnnt_amd.beam_reorder(parent, [x])[0])


@pytest.mark.parametrize("i", range(4))
def test_tracing_is_refused(i):
    """A trace would record the allocation of the results alone, and return what memory happens to hold."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = _operators()[i], torch.randn(2, 3, 8)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, x, check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(x)


def test_artefacts_built_another_way_are_stale(monkeypatch):
    """Besides their sources' times: the library's flags, and the torch and Python that the binding was compiled for."""
    import sysconfig

    from rnnt_amd import build
    _lib.native()  # builds what is missing
    assert not build.needs_build() and not build.needs_native_build()
    with monkeypatch.context() as m:
        m.setattr(build, "FLAGS", [*build.FLAGS, "-DANOTHER"])
        assert build.needs_build() and not build.needs_native_build()
    for target, name, value in ((torch, "__version__", "9.9"), (torch.version, "git_version", "0" * 40)):
        with monkeypatch.context() as m:
            m.setattr(target, name, value)
            assert build.needs_native_build() and not build.needs_build()
    with monkeypatch.context() as m:
        m.setattr(sysconfig, "get_config_var", lambda name: "another")
        assert build.needs_native_build()
    assert not build.needs_build() and not build.needs_native_build()
