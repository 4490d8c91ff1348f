"""A run of the operators as a layer uses them: rotary positions, then attention over packed documents, forward and backward, and
the same tokens one at a time behind a cache."""
import math

import pytest
import torch

from tests import dense_reference as R

pytestmark = pytest.mark.gpu


def test_embed_then_attend():
    from longcat_video_b200.modules import dense_attention, embed_rotary_qk, rotary_frequencies
    B, Hq, Hk, S, D = 1, 4, 2, 260, 64
    cu = [0, 100, 260]
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(B, S, Hq + 2 * Hk, D, generator=g, device="cuda").bfloat16().requires_grad_()
    q, k, v = (x.transpose(1, 2) for x in qkv.split([Hq, Hk, Hk], dim=2))
    f = rotary_frequencies(D, 10000.0, {"kind": "by_wavelength", "factor": 8.0, "original_length": 128})
    pos = torch.cat([torch.arange(100), torch.arange(160)]).cuda()
    qe, ke = embed_rotary_qk(q, k, f, pos)
    out = dense_attention(qe, ke, v, causal=True, softcap=15.0, cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    dout = torch.randn(out.shape, generator=g, device="cuda").bfloat16()
    (grad,) = torch.autograd.grad(out, (qkv,), dout)
    lo, hi, p = R.runs(B, S, S, True, [(cu, cu)], None, None)
    want = R.attend(qe.detach(), ke.detach(), v.detach(), lo, hi, p, 1 / math.sqrt(D), 15.0, None, dout)
    assert R.worst(out.detach(), want["o"]) <= 1
    u = 2.0 ** -8
    full = pos[None]
    parts = grad.split([Hq, Hk, Hk], dim=2)
    for part, name in zip(parts, ("dq", "dk", "dv")):
        val, bound = want[name]
        if name != "dv":  # the rotation mixes the two errors of a pair and rounds once more
            val = R.rotate(val, f.radians, f.factor, full, False, inverse=True)
            h = D // 2
            both = bound[..., :h] + bound[..., h:]
            bound = torch.cat([both, both], -1) + 2 * u * val.abs() + 2.0 ** -18
        assert R.worst(part.transpose(1, 2), (val, bound)) <= 1, name


def test_tokens_one_at_a_time():
    """A prompt read at once, then tokens behind the cache: each row is what the whole sequence gives in its place."""
    from longcat_video_b200.modules import dense_attention, embed_rotary_qk, rotary_frequencies
    B, Hq, Hk, n, total, D = 2, 8, 2, 150, 156, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(B, h, total, D, generator=g, device="cuda").bfloat16() for h in (Hq, Hk, Hk))
    f = rotary_frequencies(D)
    qe, ke = embed_rotary_qk(q, k, f)
    k_cache, v_cache = (torch.full((B, Hk, 200, D), math.nan, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    rows = []
    for a, b in [(0, n)] + [(i, i + 1) for i in range(n, total - 2)] + [(total - 2, total)]:
        qs, ks = embed_rotary_qk(q[:, :, a:b], k[:, :, a:b], f, offset=a)
        k_cache[:, :, a:b], v_cache[:, :, a:b] = ks, v[:, :, a:b]
        rows.append(dense_attention(qs, k_cache, v_cache, causal=True, k_lens=torch.full((B,), b, dtype=torch.int32, device="cuda")))
    out = torch.cat(rows, 2)
    lo, hi, p = R.runs(B, total, total, True, None, None, None)
    assert R.worst(out, R.attend(qe, ke, v, lo, hi, p, 1 / math.sqrt(D))["o"]) <= 1


@pytest.mark.parametrize("nc", [0, 2])
def test_layer_without_block_sparsity(nc):
    """self_attention with bsa_params None: RMSNorm and 3-D rotary, then every token to every token, the conditioning frames among
    themselves; the same layer with those frames cached gives the rows behind them."""
    from longcat_video_b200.modules import qk_norm_rope, self_attention, self_attention_with_kv_cache
    B, H, D, shape = 2, 3, 128, (5, 6, 7)
    N, sc = 5 * 6 * 7, nc * 6 * 7
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(B, N, 3, H, D, generator=g, device="cuda").bfloat16()
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    wq, wk = torch.rand(2, D, generator=g, device="cuda") + 0.5
    x, (k_cache, v_cache) = self_attention(q, k, v, wq, wk, shape, None, nc, return_kv=True)
    qe, ke = qk_norm_rope(q, k, wq, wk, shape)
    zero = torch.zeros(B, N, dtype=torch.int64)
    hi = torch.full((B, N), N)
    hi[:, :sc] = sc
    assert R.worst(x, R.attend(qe, ke, v, zero, hi, zero, 1 / math.sqrt(D))["o"]) <= 1
    if nc:
        new = self_attention_with_kv_cache(q[:, :, sc:], k[:, :, sc:], v[:, :, sc:], wq, wk, (5 - nc, 6, 7), (k_cache[:, :, :sc], v_cache[:, :, :sc]), None, nc)
        assert R.worst(new, tuple(t[:, :, sc:] for t in R.attend(qe, ke, v, zero, hi, zero, 1 / math.sqrt(D))["o"])) <= 1
        with pytest.raises(ValueError):
            self_attention(q, k, v, wq, wk, shape, None, 5)
