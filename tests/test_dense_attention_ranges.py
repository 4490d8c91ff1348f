"""The ends of what dense_attention takes: refusals and conversions on the host, before any launch."""
import math

import pytest
import torch

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
