"""embed_rotary and embed_rotary_qk against complex products in 64 bits.

Bound: the angle is off by 2^-24 of half a turn (its fraction rounded to 24 bits) plus sincospi's 2 steps of 2^-24, a product and a
sum in fp32 by 3 more of theirs: within 2^-20 of the pair's length; then one rounding to the type, half a step (eps / 2)."""
import pytest
import torch

from tests import dense_reference as R

pytestmark = pytest.mark.gpu


def _near(got, want, x, pairs, interleaved, factor):
    t = got.dtype
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    r = 2 * pairs
    z = x.double()
    a, b = (z[..., 0:r:2], z[..., 1:r:2]) if interleaved else (z[..., :pairs], z[..., pairs:r])
    n = torch.sqrt(a * a + b * b) * abs(factor)
    length = torch.zeros_like(z)
    if interleaved:
        length[..., 0:r:2] = length[..., 1:r:2] = n
    else:
        length[..., :pairs] = length[..., pairs:r] = n
    room = want.abs() * (torch.finfo(t).eps / 2) + length * 2.0 ** -20 * (1 + torch.finfo(t).eps) + tiny
    return bool(((got.double() - want).abs() <= room).all())


CASES = [
    # B, Hq, Hk, S, D, rotary_dim, interleaved, positions, base
    (1, 1, 1, 1, 64, 16, False, "offset", 1e4), (2, 4, 1, 1, 128, 128, False, "far", 5e5), (16, 32, 8, 1, 128, 128, True, "far", 1e4),
    (1, 3, 2, 77, 64, 64, True, "rows", 1e4), (2, 2, 2, 130, 96, 48, False, "entries", 1e4), (1, 16, 4, 1000, 128, 64, True, "rows32", 1e4),
    (1, 2, 2, 500, 256, 256, False, "offset", 1e6), (3, 5, 5, 33, 80, 32, True, "entries", 1e4), (1, 17, 1, 19, 8 * 5, 16, False, "negative", 1e4)]


def _positions(kind, B, S):
    r = torch.arange(S, device="cuda")
    if kind == "far":
        return torch.randint(2 ** 20, 2 ** 40, (B, 1), device="cuda") + r
    if kind == "rows":
        return r.flip(0) * 3
    if kind == "rows32":
        return (r + 131000).to(torch.int32)
    if kind == "entries":
        return torch.stack([r * (b + 1) for b in range(B)]).to(torch.int32 if B == 2 else torch.int64)
    if kind == "negative":
        return -r * 1001
    return None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case, dtype):
    from longcat_video_b200.modules import embed_rotary, embed_rotary_qk, rotary_frequencies
    B, Hq, Hk, S, D, rd, inter, kind, base = case
    f = rotary_frequencies(rd, base, {"kind": "by_parts", "factor": 4.0, "original_length": 4096} if S > 1 else None)
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(B, S, Hq + Hk, D, generator=g, device="cuda").to(dtype)
    q, k = qkv[:, :, :Hq].transpose(1, 2), qkv[:, :, Hq:].transpose(1, 2)
    torch.manual_seed(1)
    pos = _positions(kind, B, S)
    kw = dict(interleaved=inter) if pos is not None else dict(interleaved=inter, offset=12345)
    full = (pos if pos is not None else torch.arange(S, device="cuda") + 12345).long().expand(B, S)
    leaves = [q.detach().requires_grad_(), k.detach().requires_grad_()]
    out = embed_rotary_qk(*leaves, f, pos, **kw)
    douts = [torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in out]
    grads = torch.autograd.grad(out, leaves, douts)
    for x, y in ((q, out[0]), (k, out[1])):
        assert y.dtype == dtype and _near(y, R.rotate(x, f.radians, f.factor, full, inter), x, f.pairs, inter, f.factor)
        assert torch.equal(y[..., rd:], x[..., rd:])
        with torch.no_grad():
            assert torch.equal(embed_rotary(x, f, pos, **kw), y)
    for x, y in zip(douts, grads):
        assert _near(y, R.rotate(x, f.radians, f.factor, full, inter, inverse=True), x, f.pairs, inter, f.factor)


def test_empty_and_partial_gradients():
    from longcat_video_b200.modules import embed_rotary_qk, rotary_frequencies
    f = rotary_frequencies(32)
    q, k = torch.randn(1, 2, 6, 64, device="cuda").bfloat16(), torch.randn(1, 1, 6, 64, device="cuda").bfloat16()
    out = embed_rotary_qk(q[:, :, :0], k[:, :, :0], f)
    assert out[0].shape == (1, 2, 0, 64) and out[1].shape == (1, 1, 0, 64)
    q.requires_grad_()
    a, b = embed_rotary_qk(q, k, f, offset=3)
    (dq,) = torch.autograd.grad(a.float().square().sum(), (q,))
    # the rotation keeps lengths, so the gradient of the squared length is 2 x; four roundings to the type on the way
    assert float((dq.double() - 2 * q.detach().double()).abs().max()) <= 4 * 2.0 ** -8 * 2 * float(q.detach().abs().max()) * 2 ** 0.5


def test_captured_calls_follow_their_positions():
    from longcat_video_b200.modules import embed_rotary_qk, rotary_frequencies
    f = rotary_frequencies(64)
    q, k = torch.randn(2, 4, 9, 64, device="cuda").half(), torch.randn(2, 2, 9, 64, device="cuda").half()
    pos = torch.arange(9, device="cuda")
    embed_rotary_qk(q, k, f, pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = embed_rotary_qk(q, k, f, pos)
    pos.add_(1 << 33)
    g.replay()
    torch.cuda.synchronize()
    want = embed_rotary_qk(q, k, f, pos)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals_on_the_gpu():
    from longcat_video_b200.modules import embed_rotary, embed_rotary_qk, rotary_frequencies
    f = rotary_frequencies(64)
    x = torch.zeros(2, 2, 5, 64, device="cuda").bfloat16()
    for bad in (dict(positions=torch.zeros(4, dtype=torch.int64, device="cuda")), dict(positions=torch.zeros(5, dtype=torch.int64)),
                dict(positions=torch.zeros(5, dtype=torch.int64, device="cuda"), offset=1)):
        with pytest.raises(ValueError):
            embed_rotary(x, f, **bad)
    with pytest.raises(TypeError):
        embed_rotary(x, f, torch.zeros(5, device="cuda"))
    with pytest.raises(ValueError):
        embed_rotary(x[..., :32], f)
    from longcat_video_b200._lib import LcbsaError
    with pytest.raises(LcbsaError):
        embed_rotary_qk(x, x[:1], f)
    with pytest.raises(LcbsaError):
        embed_rotary(x.float(), f)
