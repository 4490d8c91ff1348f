"""The ends of what dense_attention takes: refusals and conversions on the host, before any launch."""
import ctypes
import math

import pytest
import torch

from longcat_video_b200 import _lib as L
from longcat_video_b200.modules import rotary_frequencies
from longcat_video_b200.modules.dense_attention import _shape_of
from tests.test_dense_attention_args import _desc, _fwd, _scores


def _shape(**kw):
    base = dict(causal=False, softcap=0.0, slopes=None, cu_q=None, cu_k=None, k_lens=None, prefix_lens=None, scale=None)
    q = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16)
    return _shape_of(q, q, **{**base, **kw})


def test_scales_that_32_bits_do_not_hold():
    """Times log2(e) a scale or a cap above 2^127.4 is infinite in 32 bits, and a score of zero NaN."""
    d = _desc(2, 4, 64, 128)
    for scale, cap in ((3e38, 0.0), (-3e38, 0.0), (3e38, 3e38), (0.0, 3e38), (2.0 ** 126, 2.0 ** 127)):
        with pytest.raises(ValueError, match="2\\^126"):
            _shape(scale=scale, softcap=cap)
        rc, msg = _fwd(d, d, d, _scores(scale=scale, cap=cap), d)
        assert rc == -1 and "2^126" in msg
    assert _shape(scale=-2.0 ** 126, softcap=2.0 ** 126)[:2] == (-2.0 ** 126, 2.0 ** 126)
    assert math.isfinite(torch.tensor(2.0 ** 126 * 1.4426950408889634, dtype=torch.float32))


def test_tangents_are_refused():
    """Before a launch, so tensors of the CPU do."""
    x = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    f = rotary_frequencies(64)
    forward = torch.autograd.forward_ad
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones_like(x))
        for i in range(3):
            qkv = [dual if j == i else x for j in range(3)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                L.binding().dense_attention(*qkv, 0.125, 0.0, False, None, None, None, None, None, False, 0)
        for xs in ((dual,), (dual, x), (x, dual)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                L.binding().rotary(xs, f.address, f.pairs, f.factor, None, 0, False)
        with pytest.raises(ValueError, match="tangent"):
            _shape(slopes=forward.make_dual(torch.ones(2), torch.ones(2)))
        assert _shape(slopes=torch.ones(2))[3].shape == (2,)


def test_numbers_that_32_bits_do_not_hold():
    """Lengths, bounds and prefixes in 64 bits are cut to what 32 hold: far behind the keys stays far behind, far before stays far before."""
    far = [-2 ** 40, -2 ** 32 + 3, 5, 2 ** 31, 2 ** 32 + 5, 2 ** 62]
    cut = [-2 ** 31, -2 ** 31, 5, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
    cu_q, cu_k = _shape(cu_q=torch.tensor(far))[4:6]
    assert cu_q.dtype == torch.int32 and cu_q.tolist() == cut and cu_k.tolist() == cut
    assert _shape(k_lens=torch.tensor([2 ** 32 + 1, -2 ** 33 + 7]))[6].tolist() == [2 ** 31 - 1, -2 ** 31]
    assert _shape(causal=True, prefix_lens=torch.tensor([[2 ** 40], [9]]))[7].tolist() == [[2 ** 31 - 1], [9]]
    same = torch.tensor([0, 4], dtype=torch.int32)
    assert _shape(cu_q=same)[4] is same
    strided = torch.arange(6, dtype=torch.int32)[::3]
    assert _shape(cu_q=strided)[4].tolist() == [0, 3] and _shape(cu_q=strided)[4].is_contiguous()


def test_a_backward_of_many_rows_needs_its_lse():
    """2^31 rows, a product that is not positive in 32 bits."""
    q, k = _desc(32768, 1, 65536, 64), _desc(32768, 1, 1, 64)
    ref = ctypes.byref
    rc = L.lib().lcbsa_dense_attn_bwd(ref(q), ref(k), ref(k), ref(q), ref(q), ref(_scores()), None, None, ref(q), ref(k), ref(k), None, 0, None)
    assert rc == -1 and "null lse" in L.lib().lcbsa_last_error().decode()
