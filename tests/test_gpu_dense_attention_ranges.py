"""dense_attention over the whole range of its arguments: values that are not finite, distances that count for a key, scales and caps at both
ends, fp16 gradients of small size.  Bounds: tests/dense_reference.py."""
import math

import pytest
import torch

from tests import dense_reference as R
from tests.test_gpu_dense_attention import MMA, TC, _dense, _inputs, _slopes

pytestmark = pytest.mark.gpu


# ---- values that are not finite where nothing sees them ----------------------------------------------------------------------------

@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_documents_keep_their_gradients_apart(cap, poison, D, dtype):
    """q, k, v and dout of the rows before the first document and behind the last, and of a whole document in between, hold NaN or infinities:
    outputs and gradients of the documents beside them stay within their bounds, the gradients of rows of no document are zero."""
    S, cu = 420, [20, 150, 290, 400]
    q, k, v, dout = _inputs(1, 4, 2, S, S, D, dtype, seed=20)
    lo, hi, pos = R.runs(1, S, S, True, [(cu, cu)], None, None)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), cap, None, dout)
    for x in (q, k, v, dout):
        x[:, :, :20] = x[:, :, 400:] = x[:, :, 150:290] = poison
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, causal=True, softcap=cap, cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    grads = torch.autograd.grad(out, leaves, dout)
    rows = [*range(20, 150), *range(290, 400)]
    outside = [*range(20), *range(400, S)]
    for got, x in zip((out.detach(), *grads), ("o", "dq", "dk", "dv")):
        val, bound = want[x]
        assert R.worst(got[:, :, rows], (val[:, :, rows], bound[:, :, rows])) <= 1, x
        assert not got[:, :, outside].any(), x


# ---- slopes below zero -------------------------------------------------------------------------------------------------------------

NEGATIVE = {  # the last unit of 64 queries is not full, and keys far from it are seen by all of its queries
    "all_seen": ((1, 4, 2, 330, 330), dict()),
    "all_seen_short": ((2, 2, 2, 100, 100), dict()),
    "causal": ((1, 4, 2, 330, 330), dict(causal=True)),
    "causal_prefix": ((1, 2, 1, 290, 290), dict(causal=True, prefix=[[200]])),
    "one_query": ((2, 4, 2, 1, 300), dict()),
    "documents": ((1, 2, 2, 415, 415), dict(docs=[([0, 60, 415], [0, 60, 415])])),
}


@pytest.mark.parametrize("impl", [TC, MMA])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("name", NEGATIVE)
def test_slopes_below_zero(name, D, dtype, cap, impl):
    """A distance that counts for a key: far keys weigh most.  x is at most 40 + 0.5 * 415 in size, so the distance in fp32 is off by 2^-24 of 250,
    1.5e-5, which SCORE has room for."""
    (B, Hq, Hk, Sq, Sk), o = NEGATIVE[name]
    docs, prefix, causal = o.get("docs"), o.get("prefix"), o.get("causal", False)
    lo, hi, pos = R.runs(B, Sq, Sk, causal, docs, None, prefix)
    slopes = -_slopes(Hq)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kw = dict(causal=causal, softcap=cap, slopes=slopes, impl=impl)
    if docs:
        kw["cu_q"], kw["cu_k"] = ints(docs[0][0]), ints(docs[0][1])
    if prefix:
        kw["prefix_lens"] = ints(prefix[0])
    q, k, v, dout = _inputs(B, Hq, Hk, Sq, Sk, D, dtype, seed=21)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), cap, slopes, dout)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, dout)
    for got, x in zip((out.detach(), *grads), ("o", "dq", "dk", "dv")):
        assert R.worst(got, want[x]) <= 1, x


# ---- scales and caps at both ends of what is accepted ------------------------------------------------------------------------------

@pytest.mark.parametrize("impl", [TC, MMA])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale,cap", [(2.0 ** 20, 1.0), (-2.0 ** 20, 1.0), (4096.0, 2.0 ** -8), (2.0 ** 40, 2.0 ** 22), (2.0 ** 90, 4.0 * 2.0 ** 70),
                                       (1.0, 2.0 ** 20), (2.0 ** -4, 2.0 ** 16), (2.0 ** -40, 2.0 ** -20)])
def test_scales_far_from_their_cap(scale, cap, D, impl):
    """Scores of some units of the cap or of one, whichever is less, among them rows and keys of zeros: the formulas' bounds, whatever powers of
    scale and cap come to in 32 bits.  The inputs keep sums of |q_d k_d| scale below 40: q is 2^e / scale times a normal number."""
    B, Hq, Hk, S = 1, 4, 2, 150
    q, k, v, dout = _inputs(B, Hq, Hk, S, S, D, torch.bfloat16, seed=22)
    size = min(1.0, 4 * cap) * (0.5 if D == 64 else 0.25)
    q = (q.float() * (size / abs(scale))).bfloat16()
    q[:, :, 10:20] = 0
    k[:, :, 30:35] = 0
    q[:, :, 140] *= 2.0 ** -6
    lo, hi, pos = R.runs(B, S, S, True, None, None, None)
    want = R.attend(q, k, v, lo, hi, pos, scale, cap, None, dout)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out, lse = _dense()(*leaves, causal=True, scale=scale, softcap=cap, return_lse=True, impl=impl)
    assert R.worst(out.detach(), want["o"]) <= 1
    assert float((lse.double() - want["lse"]).abs().max()) <= R.SCORE + 1e-5
    for got, x in zip(torch.autograd.grad(out, leaves, dout), ("dq", "dk", "dv")):
        assert R.worst(got, want[x]) <= 1, x


# ---- values that are not finite in one operand alone -------------------------------------------------------------------------------

@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("poison", [math.inf, math.nan])
def test_values_do_not_reach_their_own_gradient(poison, D, dtype):
    """dv is P^T dout: infinities and NaN in v, which make outputs and dq of the rows that see them what they are, leave dv alone, in tiles that all
    rows see and in those that some see."""
    S = 400
    q, k, v, dout = _inputs(1, 4, 2, S, S, D, dtype, seed=23)
    lo, hi, pos = R.runs(1, S, S, True, None, None, None)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), 0.0, None, dout)["dv"]
    v[0, 1, 40, 5] = v[0, 0, 333, 7] = poison
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, causal=True)
    assert not torch.isfinite(out[0, 2, 40:, 5]).any()
    assert R.worst(torch.autograd.grad(out, leaves, dout)[2], want) <= 1


@pytest.mark.parametrize("poison", [math.inf, -math.inf, math.nan])
def test_a_gradient_that_is_not_finite_stays_with_its_row(poison):
    """dout of one query of one head, in one dimension: dv of the keys that it sees is not finite there, of all others it is within its bound; dq of
    the other rows too."""
    S, D, i, c = 400, 128, 211, 9
    q, k, v, dout = _inputs(1, 2, 2, S, S, D, torch.bfloat16, seed=24)
    lo, hi, pos = R.runs(1, S, S, True, None, None, None)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), 0.0, None, dout)
    dout[0, 1, i, c] = poison
    leaves = [x.requires_grad_() for x in (q, k, v)]
    dq, _, dv = torch.autograd.grad(_dense()(*leaves, causal=True), leaves, dout)
    assert not torch.isfinite(dv[0, 1, :i + 1, c]).any()
    part = lambda x, idx: tuple(t[idx] for t in x)  # noqa: E731
    assert R.worst(dv[0, 0], part(want["dv"], (0, 0))) <= 1 and R.worst(dv[0, 1, i + 1:], part(want["dv"], (0, 1, slice(i + 1, None)))) <= 1
    rows = [r for r in range(S) if r != i]
    assert R.worst(dq[0, 1, rows], part(want["dq"], (0, 1, rows))) <= 1
    assert not torch.isfinite(dq[0, 1, i]).any()


# ---- hidden values under a cap -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("poison", [math.inf, -math.inf, math.nan, 3e4])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("D,Sq,impl", [(128, 6, MMA), (128, 200, MMA), (128, 200, TC), (64, 200, TC)])
def test_hidden_keys_under_a_cap(D, Sq, impl, slopes, poison):
    """What keys behind the length hold, numbers far beyond the cap among them, changes not a bit of outputs and gradients."""
    B, Hq, Hk, Sk = 2, 4, 2, 300
    q, k, v, dout = _inputs(B, Hq, Hk, Sq, Sk, D, torch.float16, seed=25)
    lens = torch.tensor([200 + Sq % 7, 61], dtype=torch.int32, device="cuda")
    kw = dict(causal=True, k_lens=lens, softcap=30.0, slopes=_slopes(Hq) if slopes else None, impl=impl)

    def all_of(k, v):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, **kw)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    kp, vp = k.clone(), v.clone()
    for b in range(B):
        kp[b, :, int(lens[b]):] = poison
        vp[b, :, int(lens[b]):] = poison
    assert all(torch.equal(a, b) for a, b in zip(all_of(kp, vp), all_of(k, v)))


@pytest.mark.parametrize("poison", [math.nan, 3e4])
def test_later_keys_under_a_cap(poison):
    """What comes behind a query in the order changes not a bit of its output: its neighbours, which see it, may be NaN or at the cap."""
    S = 300
    q, k, v, _ = _inputs(1, 4, 2, S, S, 128, torch.float16, seed=26)
    for slopes in (None, _slopes(4)):
        call = lambda k, v: _dense()(q, k, v, causal=True, softcap=30.0, slopes=slopes, impl=TC)  # noqa: E731
        want = call(k, v)
        kp, vp = k.clone(), v.clone()
        kp[:, :, 150:152] = poison
        vp[:, :, 150:152] = poison
        assert torch.equal(call(kp, vp)[:, :, :150], want[:, :, :150])


# ---- fp16 gradients of small size --------------------------------------------------------------------------------------------------

def test_small_fp16_gradients_are_kept():
    """256 keys of equal weight (q or k zero), values of +-1, dout 2^-16 in one dimension: dS is +-2^-24 before the factor scale = 1/8, the smallest
    number that fp16 has, and nothing behind it.  dq and dk are 256 * 2^-27 = 2^-19.  P and dS are off by a few 2^-24 of their size (lse, ex2), so dS
    rounds to +-2^-24, and the sums are exact but for that: the result is 2^-19, on the grid of fp16."""
    n, D = 256, 64
    sign = 1.0 - 2.0 * (torch.arange(n, device="cuda") % 2)
    zero = lambda: torch.zeros(1, 1, n, D, device="cuda", dtype=torch.float16)  # noqa: E731
    for side in ("dq", "dk"):
        q, k, v, dout = zero(), zero(), zero(), zero()
        v[0, 0, :, 0] = sign.half()
        dout[..., 0] = 2.0 ** -16
        (k if side == "dq" else q)[0, 0, :, 3] = sign.half() if side == "dq" else 1.0
        leaves = [x.requires_grad_() for x in (q, k, v)]
        dq, dk, _ = torch.autograd.grad(_dense()(*leaves), leaves, dout)
        want = zero()
        want[0, 0, :, 3] = 2.0 ** -19 if side == "dq" else (sign * 2.0 ** -19).half()
        assert torch.equal(dq if side == "dq" else dk, want), side


@pytest.mark.parametrize("scale", [None, -0.05])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3])
@pytest.mark.parametrize("D,heads", [(64, (2, 2)), (128, (8, 2))])
def test_roundings_of_small_fp16_gradients(D, heads, size, scale):
    """The root mean square error of dq and dk against that of independent roundings: each dS / scale off by a uniform error of one step of fp16 at its
    size (step / sqrt(12), 2^-24 at least), times scale and the other operand; the result off by half of its own step.  delta and P, whose errors are
    2^-20 and less of a dS, have the rest of the factor 1.25 (the two groups of errors, at sizes 1 to 1e-3, are 10^4 numbers and more)."""
    B, S, (Hq, Hk) = 1, 1500, heads
    q, k, v, dout = _inputs(B, Hq, Hk, S, S, D, torch.float16, seed=27)
    dout = (dout.float() * size).half()
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(_dense()(*leaves, scale=scale), leaves, dout)
    scale = D ** -0.5 if scale is None else scale
    step = lambda x: torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14))) - 10)  # noqa: E731
    G = Hq // Hk
    kk, vv = k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    p = torch.softmax(q.double() @ kk.transpose(-1, -2) * scale, -1)
    dp = dout.double() @ vv.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    var = (step(ds) * scale) ** 2 / 12
    fold = lambda x: x.view(B, Hk, G, S, D).sum(2)  # noqa: E731
    for got, want, v2 in ((dq, ds @ kk * scale, var @ kk ** 2), (dk, fold(ds.transpose(-1, -2) @ q.double()) * scale, fold(var.transpose(-1, -2) @ q.double() ** 2))):
        room = 1.25 * (v2 + step(want) ** 2 / 12).mean().sqrt()
        assert float((got.double() - want).square().mean().sqrt()) <= float(room)


# ---- forward-mode derivatives ------------------------------------------------------------------------------------------------------

def test_tangents_are_refused():
    """A tangent that no rule carries on is an error, with and without a backward recorded; outside of its level the call goes through."""
    from longcat_video_b200.modules import embed_rotary, embed_rotary_qk, rotary_frequencies
    q, k, v, _ = _inputs(1, 2, 2, 20, 20, 64, torch.bfloat16)
    f = rotary_frequencies(64)
    with torch.autograd.forward_ad.dual_level():
        for grad in (False, True):
            dual = torch.autograd.forward_ad.make_dual(q.clone().requires_grad_(grad), torch.ones_like(q))
            for call in (lambda: _dense()(dual, k, v), lambda: _dense()(q, dual, v), lambda: _dense()(q, k, dual), lambda: embed_rotary(dual, f),
                         lambda: embed_rotary_qk(q, dual, f)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        assert torch.equal(_dense()(q, k, v), _dense()(q, k, v))


# ---- numbers that 32 bits do not hold ----------------------------------------------------------------------------------------------

def test_lengths_beyond_32_bits():
    q, k, v, _ = _inputs(1, 2, 2, 30, 90, 64, torch.bfloat16)
    far = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    for impl in (TC, MMA):
        assert torch.equal(_dense()(q, k, v, k_lens=far(2 ** 32 + 5), impl=impl), _dense()(q, k, v, impl=impl))
        assert torch.equal(_dense()(q, k, v, k_lens=far(-2 ** 33 + 50), impl=impl), torch.zeros_like(q))
        assert torch.equal(_dense()(q, k, v, causal=True, prefix_lens=far(2 ** 40), impl=impl), _dense()(q, k, v, impl=impl))


def test_a_document_far_before_the_queries():
    """Its end is the lowest number of 32 bits: nothing of it is in the tensor, and the keys of the document behind it, in the same unit of 64 as its own,
    have their gradients."""
    q, k, v, dout = _inputs(1, 2, 2, 600, 400, 64, torch.bfloat16)  # query 210 is the first to see key 10, 264 key 64: units 3 and 4
    cu_k = torch.tensor([0, 10, 400], dtype=torch.int32, device="cuda")

    def grads(first):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        cu_q = torch.tensor([first, first, 600], dtype=torch.int32, device="cuda")
        return torch.autograd.grad(_dense()(*leaves, causal=True, cu_q=cu_q, cu_k=cu_k), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads(-2 ** 31), grads(0)))


@pytest.mark.parametrize("impl", [TC, MMA])
def test_bounds_beyond_the_tensors_under_an_order(impl):
    """Documents that reach beyond the tensors are cut at their ends before anything is counted from these: the last query there is stands at the last
    key there is."""
    q, k, v, dout = _inputs(2, 4, 2, 150, 230, 128, torch.bfloat16, seed=28)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def all_of(cu_q, cu_k, **kw):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True, cu_q=ints(*cu_q), cu_k=ints(*cu_k), impl=impl, **kw)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    for kw in (dict(), dict(slopes=_slopes(4)), dict(prefix_lens=ints(30, 90), softcap=10.0)):
        want = all_of((0, 60, 150), (0, 100, 230), **kw)
        for cu_q, cu_k in (((0, 60, 178), (0, 100, 230)), ((-30, 60, 2 ** 31 - 1), (-5, 100, 231)), ((0, 60, 150), (-2 ** 31, 100, 2 ** 31 - 1))):
            assert all(torch.equal(a, b) for a, b in zip(all_of(cu_q, cu_k, **kw), want))
