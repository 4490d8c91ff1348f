"""Refusals of dense_attention and the 1-D rotary embedding, and the frequencies: on the host, before any launch."""
import ctypes
import math

import pytest
import torch

from longcat_video_b200 import _lib as L
from longcat_video_b200.modules import dense_attention, embed_rotary, rotary_frequencies
from longcat_video_b200.modules.dense_attention import _shape_of


def _desc(B, H, S, D, dtype=L.LCBSA_BF16, data=4096):
    t = L.LcbsaTensor()
    t.data, t.dtype = data, dtype
    for i, (n, s) in enumerate(zip((B, H, S, D), (H * S * D, S * D, D, 1))):
        t.size[i], t.stride[i] = n, s
    return t


def _scores(**kw):
    s = L.LcbsaScores()
    s.scale = 0.1
    for n, x in kw.items():
        setattr(s, n, x)
    return s


def _fwd(q, k, v, s, out, ws=None, n=0):
    ref = ctypes.byref
    return L.lib().lcbsa_dense_attn_fwd(ref(q), ref(k), ref(v), ref(s), ref(out), None, None, ws, n, None), L.lib().lcbsa_last_error().decode()


def test_no_cpu_path():
    x = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        dense_attention(x, x, x)
    with pytest.raises(RuntimeError):
        embed_rotary(x, rotary_frequencies(64))


@pytest.mark.parametrize("kw", [
    dict(softcap=-1.0), dict(softcap=math.inf), dict(scale=math.nan), dict(cu_k=torch.tensor([0, 4])), dict(cu_q=torch.tensor([0])),
    dict(cu_q=torch.tensor([0, 4]), k_lens=torch.tensor([4, 4])), dict(cu_q=torch.tensor([0, 4]), cu_k=torch.tensor([0, 2, 4])),
    dict(cu_q=torch.zeros(3, 2, dtype=torch.int32)), dict(k_lens=torch.tensor([4])), dict(prefix_lens=torch.tensor([1])),
    dict(prefix_lens=torch.tensor([1, 2]), causal=True, cu_q=torch.tensor([0, 4])), dict(slopes=torch.ones(3)),
    dict(slopes=torch.ones(2, requires_grad=True))])
def test_shapes_are_checked(kw):
    q = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16)
    base = dict(causal=False, softcap=0.0, slopes=None, cu_q=None, cu_k=None, k_lens=None, prefix_lens=None, scale=None)
    with pytest.raises(ValueError):
        _shape_of(q, q, **{**base, **kw})
    with pytest.raises(TypeError):
        _shape_of(q, q, **{**base, "k_lens": torch.ones(2)})


def test_a_cap_far_from_the_scale_is_refused():
    q = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16)
    for cap, scale, ok in ((131072.0, None, True), (131073.0, None, False), (1e-7, None, False), (1.0, -2.0 ** 20, True), (1.0, 2.0 ** -21, False), (5.0, 0.0, True)):
        if ok:
            assert _shape_of(q, q, False, cap, None, None, None, None, None, scale)[1] == cap
        else:
            with pytest.raises(ValueError, match="2\\^20"):
                _shape_of(q, q, False, cap, None, None, None, None, None, scale)
    d = _desc(2, 4, 64, 128)
    rc, msg = _fwd(d, d, d, _scores(scale=1.0, cap=2e6), d)
    assert rc == -1 and "2^20" in msg


def test_scalings_name_what_is_missing():
    from longcat_video_b200.modules import rotary_frequencies
    for scaling in ({"kind": "by_parts", "factor": 4.0}, {"kind": "by_wavelength", "factor": 4.0, "original_length": 0}, {"kind": "linear", "factor": math.inf}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, 10000.0, scaling)


def test_the_library_refuses_before_a_launch():
    q, k = _desc(2, 4, 64, 128), _desc(2, 2, 100, 128)
    ok = _scores()
    for args, word in (((q, k, _desc(2, 2, 101, 128), ok, q), "different shapes"), ((q, _desc(2, 3, 100, 128), _desc(2, 3, 100, 128), ok, q), "evenly"),
                       ((q, _desc(1, 2, 100, 128), _desc(1, 2, 100, 128), ok, q), "disagree"), ((q, k, k, ok, k), "another shape"),
                       ((q, k, k, _scores(cap=-1.0), q), "cap"), ((q, k, k, _scores(scale=math.inf), q), "finite"),
                       ((q, k, k, _scores(cu_q=4096), q), "go together"), ((q, k, k, _scores(cu_q=4096, cu_k=4096), q), "at least 1"),
                       ((q, k, k, _scores(cu_q=4096, cu_k=4096, docs=1, k_len=4096), q), "exclude"), ((q, k, k, _scores(prefix=4096), q), "causal"), ((q, k, k, _scores(impl=3), q), "impl"),
                       ((_desc(2, 4, 64, 128, data=4100), k, k, ok, q), "16-byte"), ((_desc(2, 4, 64, 128, L.LCBSA_FP16), k, k, ok, q), "dtypes")):
        rc, msg = _fwd(*args)
        assert rc == -1 and word in msg, msg
    d96 = _desc(1, 1, 8, 96)
    assert _fwd(d96, d96, d96, ok, d96)[0] == -2
    f32 = _desc(1, 1, 8, 64, L.LCBSA_FP32)
    assert _fwd(f32, f32, f32, ok, f32)[0] == -2
    ref = ctypes.byref
    rc = L.lib().lcbsa_dense_attn_bwd(ref(q), ref(k), ref(k), ref(q), ref(q), ref(ok), 4096, None, ref(q), ref(k), ref(k), None, 0, None)
    assert rc == -3
    rc = L.lib().lcbsa_dense_attn_bwd(ref(q), ref(k), ref(k), ref(q), ref(q), ref(ok), None, None, ref(q), ref(k), ref(k), 4096, 1 << 30, None)
    assert rc == -1


def test_rotary_refusals():
    x, y = _desc(1, 2, 8, 64), _desc(1, 2, 8, 64)
    f = rotary_frequencies(64)
    ref = ctypes.byref
    call = lambda x, y, n, pairs, bits=64, pos=4096, factor=1.0: L.lib().lcbsa_rotary(  # noqa: E731
        ref(x), ref(y), n, f.turns, pairs, 0, 0, factor, pos, bits, 0, 1, 0, None)
    assert call(x, y, 0, 32) == -1 and call(x, y, 3, 32) == -1
    for pairs in (0, 4, 12, 40, 136):  # 40: more than half of the head
        assert call(x, y, 1, pairs) == -1
    assert call(x, y, 1, 32, bits=16) == -1 and call(x, y, 1, 32, factor=math.nan) == -1
    assert call(x, _desc(1, 2, 9, 64), 1, 32) == -1 and call(x, _desc(1, 2, 8, 64, L.LCBSA_FP16), 1, 32) == -1
    assert call(_desc(1, 2, 8, 64, L.LCBSA_FP32), y, 1, 32) == -2
    for kw in (dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=272), dict(rotary_dim=64, base=1.0),
               dict(rotary_dim=64, scaling={"kind": "other", "factor": 2.0}), dict(rotary_dim=64, scaling={"kind": "linear", "factor": 0.5}),
               dict(rotary_dim=64, scaling={"kind": "linear", "factor": 2.0, "original_length": 10}),
               dict(rotary_dim=64, scaling={"kind": "by_wavelength", "factor": 2.0, "original_length": 10, "low": 4.0, "high": 4.0})):
        with pytest.raises(ValueError):
            rotary_frequencies(**kw)


def test_frequencies():
    """Turns are the radians over 2 pi as 64-bit fractions; the scalings at their ends."""
    f = rotary_frequencies(64, 10000.0)
    assert f.pairs == 32 and f.factor == 1.0
    for i in range(32):
        assert f.radians[i] == pytest.approx(10000.0 ** (-2 * i / 64), rel=1e-14)
        assert abs(f.turns[i] / 2 ** 64 - f.radians[i] / (2 * math.pi)) <= 2 ** -54  # the division by 2 pi here
    lin = rotary_frequencies(64, 10000.0, {"kind": "linear", "factor": 4.0})
    assert all(a == pytest.approx(b / 4) for a, b in zip(lin.radians, f.radians))
    base = rotary_frequencies(64, 10000.0, {"kind": "base", "factor": 4.0})
    assert base.radians[0] == 1.0 and base.radians[-1] == pytest.approx(f.radians[-1] / 4)
    parts = rotary_frequencies(64, 10000.0, {"kind": "by_parts", "factor": 16.0, "original_length": 4096})
    assert parts.radians[0] == f.radians[0] and parts.radians[-1] == pytest.approx(f.radians[-1] / 16)
    assert parts.factor == pytest.approx(0.1 * math.log(16) + 1)
    wave = rotary_frequencies(64, 10000.0, {"kind": "by_wavelength", "factor": 8.0, "original_length": 4096})
    assert wave.radians[0] == f.radians[0] and wave.radians[-1] == pytest.approx(f.radians[-1] / 8) and wave.factor == 1.0
    assert rotary_frequencies(64) is f
