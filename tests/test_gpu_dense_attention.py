"""dense_attention against the formulas in 64 bits: outputs, log-sum-exp and gradients, with bounds from the roundings made
(tests/dense_reference.py), at the sizes and masks where it can go wrong."""
import math

import pytest
import torch

from tests import dense_reference as R

pytestmark = pytest.mark.gpu


def _dense():
    from longcat_video_b200.modules import dense_attention
    return dense_attention


def _inputs(B, Hq, Hk, Sq, Sk, D, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v, dout = new(B, Hq, Sq, D) * spread, new(B, Hk, Sk, D), new(B, Hk, Sk, D), new(B, Hq, Sq, D)
    return [x.to(dtype) for x in (q, k, v, dout)]


def _slopes(Hq):
    return 0.5 ** (1 + torch.arange(Hq, device="cuda", dtype=torch.float32) * 8 / Hq)


CASES = {
    # name: (B, Hq, Hk, Sq, Sk), options; docs: per entry (cu_q, cu_k)
    "one_token": ((2, 8, 2, 1, 1), {}),
    "one_token_cache": ((3, 8, 2, 1, 777), dict(k_lens=[777, 1, 300], causal=True)),
    "empty_cache": ((3, 4, 4, 1, 200), dict(k_lens=[0, 200, 64], causal=True)),
    "drafts": ((2, 12, 2, 5, 333), dict(k_lens=[333, 129], causal=True, slopes=True)),
    "drafts_before_keys": ((2, 4, 2, 7, 40), dict(k_lens=[3, 40], causal=True)),  # the first queries stand before the first key
    "square": ((2, 2, 2, 64, 64), {}),
    "odd": ((1, 3, 1, 77, 131), dict(cap=20.0)),
    "causal_odd": ((1, 4, 2, 193, 193), dict(causal=True, cap=5.0)),
    "causal_longer_keys": ((1, 2, 1, 100, 301), dict(causal=True, slopes=True)),
    "causal_longer_queries": ((1, 2, 1, 301, 100), dict(causal=True)),  # 201 queries see nothing
    "prefix": ((2, 2, 2, 200, 200), dict(causal=True, prefix=[[70], [0]], slopes=True)),
    "prefix_beyond": ((1, 2, 2, 90, 90), dict(causal=True, prefix=[[1000]])),
    "documents": ((1, 4, 2, 300, 300), dict(causal=True, docs=[([0, 1, 64, 64, 190, 300], None)], cap=30.0)),
    "documents_bidirectional": ((1, 2, 2, 260, 260), dict(docs=[([0, 5, 133, 260], None)], slopes=True)),
    "documents_tail": ((1, 2, 2, 260, 260), dict(docs=[([10, 100, 200], None)], causal=True)),  # rows of no document on both sides
    "documents_prefix": ((1, 2, 1, 260, 260), dict(docs=[([0, 100, 260], None)], causal=True, prefix=[[30, 100]])),
    "documents_per_entry": ((2, 2, 2, 150, 150), dict(docs=[([0, 50, 150], None), ([0, 149, 150], None)])),
    "cross": ((1, 4, 4, 400, 100), dict(docs=[([0, 130, 400], [0, 33, 100])])),
    "cross_empty_text": ((1, 2, 2, 200, 70), dict(docs=[([0, 90, 150, 200], [0, 40, 40, 70])])),
    "long": ((1, 2, 1, 1100, 1100), dict(causal=True, cap=50.0, slopes=True)),
    "long_keys": ((1, 4, 2, 130, 2500), {}),
    "wide_scores": ((1, 2, 2, 150, 150), dict(spread=6.0, scale=0.05, causal=True)),
    "negative_scale": ((1, 2, 2, 100, 100), dict(scale=-0.1, cap=3.0)),
}


def _options(case, dtype, D):
    (B, Hq, Hk, Sq, Sk), o = case
    docs = o.get("docs")
    if docs is not None:
        docs = [(cq, cq if ck is None else ck) for cq, ck in docs]
        docs = docs * B if len(docs) == 1 else docs
    lo, hi, pos = R.runs(B, Sq, Sk, o.get("causal", False), docs, o.get("k_lens"), o.get("prefix") and o["prefix"] * (B if len(o["prefix"]) == 1 else 1))
    kw = dict(causal=o.get("causal", False), softcap=o.get("cap", 0.0), scale=o.get("scale"))
    if o.get("slopes"):
        kw["slopes"] = _slopes(Hq)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if docs is not None:
        kw["cu_q"], kw["cu_k"] = ints([d[0] for d in docs]), ints([d[1] for d in docs])
        if len(o["docs"]) == 1:
            kw["cu_q"], kw["cu_k"] = kw["cu_q"][0], kw["cu_k"][0]
    if "k_lens" in o:
        kw["k_lens"] = ints(o["k_lens"])
    if "prefix" in o:
        kw["prefix_lens"] = ints(o["prefix"] if len(o["prefix"]) == B else o["prefix"][0])
    return lo, hi, pos, kw, o.get("scale") or 1 / math.sqrt(D), o.get("spread", 1.0)


TC, MMA = 1, 2  # the forward kernels: tcgen05, and the one for few queries


@pytest.mark.parametrize("impl", [TC, MMA])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("name", CASES)
def test_forward_and_gradients(name, D, dtype, impl):
    B, Hq, Hk, Sq, Sk = CASES[name][0]
    lo, hi, pos, kw, scale, spread = _options(CASES[name], dtype, D)
    q, k, v, dout = _inputs(B, Hq, Hk, Sq, Sk, D, dtype, spread=spread)
    want = R.attend(q, k, v, lo, hi, pos, scale, kw["softcap"], kw.get("slopes"), dout)
    with torch.no_grad():
        plain, lse = _dense()(q, k, v, return_lse=True, impl=impl, **kw)
    assert R.worst(plain, want["o"]) <= 1
    blind = torch.isinf(want["lse"])
    assert torch.equal(torch.isinf(lse), blind) and torch.equal(plain[blind], torch.zeros_like(plain[blind]))
    assert float((lse.double() - want["lse"])[~blind].abs().max()) <= R.SCORE + 1e-5
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, impl=impl, **kw)
    grads = torch.autograd.grad(out, leaves, dout)
    assert torch.equal(out, plain)
    for got, x in zip(grads, ("dq", "dk", "dv")):
        assert got.dtype == dtype and R.worst(got, want[x]) <= 1, x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_against_differences(dtype):
    """The directional derivative of sum(w o) from the formula's gradients (which the kernel is held to elsewhere) and the
    kernel's own, against a central difference of the function in 64 bits."""
    B, Hq, Hk, S, D = 1, 2, 1, 90, 64
    q, k, v, w = _inputs(B, Hq, Hk, S, S, D, dtype, seed=3)
    lo, hi, pos = R.runs(B, S, S, True, None, None, [[20]])
    kw = dict(causal=True, softcap=4.0, slopes=_slopes(Hq), prefix_lens=torch.tensor([20], dtype=torch.int32, device="cuda"))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(_dense()(*leaves, **kw), leaves, w)
    want = R.attend(q, k, v, lo, hi, pos, 1 / 8, 4.0, kw["slopes"], w)
    g = torch.Generator(device="cuda").manual_seed(5)
    for x in range(3):
        step = torch.randn(leaves[x].shape, generator=g, device="cuda", dtype=torch.float64)
        vals = []
        for sign in (1, -1):
            moved = [t.double() for t in (q, k, v)]
            moved[x] = moved[x] + sign * 1e-5 * step
            vals.append(float((_in_64(moved, lo, hi, pos, 1 / 8, 4.0, kw["slopes"]) * w.double()).sum()))
        slope = (vals[0] - vals[1]) / 2e-5
        room = float((want[("dq", "dk", "dv")[x]][1] * step.abs()).sum())
        assert abs(float((grads[x].double() * step).sum()) - slope) <= room


def _in_64(qkv, lo, hi, pos, scale, cap, slopes):
    q, k, v = qkv
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    j = torch.arange(k.shape[2], device=q.device)
    lo, hi, pos = (x.to(q.device)[:, None, :, None] for x in (lo, hi, pos))
    s = cap * torch.tanh(q @ k.transpose(-1, -2) * scale / cap) - slopes.double()[None, :, None, None] * (pos - j).abs()
    return torch.softmax(s.masked_fill((j < lo) | (j >= hi), -math.inf), -1) @ v


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Sq,impl", [(1, MMA), (6, MMA), (200, MMA), (200, TC), (3, TC)])
def test_hidden_keys_may_hold_anything(poison, Sq, impl):
    """Keys behind the length, keys of another document, queries of no document: not a bit of the result changes."""
    B, Hq, Hk, Sk, D = 2, 4, 2, 300, 128
    q, k, v, dout = _inputs(B, Hq, Hk, Sq, Sk, D, torch.bfloat16, seed=1)
    lens = torch.tensor([200 + Sq % 7, 61], dtype=torch.int32, device="cuda")
    kw = dict(causal=True, k_lens=lens, impl=impl)

    def all_of(q, k, v):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, **kw)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    clean = all_of(q, k, v)
    kp, vp = k.clone(), v.clone()
    for b in range(B):
        kp[b, :, int(lens[b]):] = poison
        vp[b, :, int(lens[b]):] = poison
    for got, want in zip(all_of(q, kp, vp), clean):
        assert torch.equal(got, want)


@pytest.mark.parametrize("D,dtype,impl", [(128, torch.bfloat16, TC), (64, torch.float16, TC), (128, torch.bfloat16, MMA)])
def test_documents_and_order_keep_values_apart(D, dtype, impl):
    """One document, and the later half of another, hold NaN and infinities in q, k, v and dout: the results of the rows that do not see
    them, and the gradients of the keys that are not seen by such queries, are finite and within their bounds."""
    S, H = 400, 2
    cu = [0, 150, 290, 400]
    q, k, v, dout = _inputs(1, H, 1, S, S, D, dtype, seed=2)
    lo, hi, pos = R.runs(1, S, S, True, [(cu, cu)], None, None)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), 0.0, None, dout)
    bad = {150, 163, 251, 350, 399}  # document 1 from its first token on, document 2 from token 350 on
    for x in (q, k, v, dout):
        for n, i in enumerate(sorted(bad)):
            x[0, :, i, (7 * n) % D] = (math.nan, math.inf, -math.inf)[n % 3]
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, causal=True, cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"), impl=impl)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    rows = list(range(0, 150)) + list(range(290, 350))  # see no bad key
    keys = list(range(0, 150))                            # seen by no bad query
    for got, x, idx in ((out, "o", rows), (dq, "dq", rows), (dk, "dk", keys), (dv, "dv", keys)):
        val, bound = want[x]
        assert R.worst(got[:, :, idx], (val[:, :, idx], bound[:, :, idx])) <= 1, x
    assert torch.isnan(out[:, :, 150:290]).any(-1).all() and torch.isnan(dq[:, :, 150:290]).any(-1).all()


@pytest.mark.parametrize("impl", [TC, MMA])
def test_a_seen_infinity_stays_where_it_is(impl):
    """v = inf in one dimension of a key that some rows of a tile see: those rows are inf there and finite elsewhere."""
    q, k, v, _ = _inputs(1, 2, 2, 100, 100, 64, torch.bfloat16, seed=4)
    v[0, 1, 40, 5] = math.inf
    out = _dense()(q, k, v, causal=True, impl=impl)
    assert torch.isposinf(out[0, 1, 40:, 5]).all()
    out[0, 1, 40:, 5] = 0
    assert torch.isfinite(out).all()
    q1 = q[:, :, :1]
    out = _dense()(q1, k, v, k_lens=torch.tensor([41], dtype=torch.int32, device="cuda"), impl=impl)
    assert torch.isposinf(out[0, 1, 0, 5]) and int(torch.isfinite(out).sum()) == out.numel() - 1


@pytest.mark.parametrize("impl", [TC, MMA])
def test_a_nan_score_makes_its_rows_nan(impl):
    q, k, v, _ = _inputs(1, 2, 2, 130, 130, 64, torch.bfloat16, seed=4)
    k[0, 0, 70, 3] = math.nan
    out, lse = _dense()(q, k, v, causal=True, return_lse=True, impl=impl)
    assert torch.isnan(out[0, 0, 70:]).all() and torch.isfinite(out[0, 0, :70]).all() and torch.isfinite(out[0, 1]).all()
    assert torch.isnan(lse[0, 0, 70:]).all() and torch.isfinite(lse[0, 0, :70]).all()


def test_strides_and_broadcast():
    """Views of a fused projection, a key cache longer than what is used, one cache for all entries: the bits of contiguous copies; the
    gradient of the shared cache is the sum over the entries."""
    B, Hq, Hk, S, D = 2, 4, 2, 150, 128
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(B, S, Hq + 2 * Hk, D, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = (x.transpose(1, 2) for x in qkv.split([Hq, Hk, Hk], dim=2))
    want = _dense()(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(_dense()(q, k, v, causal=True), want)
    odd = torch.randn(B, Hq, S, D + 1, generator=g, device="cuda").to(torch.bfloat16)[..., 1:]  # neither aligned nor a legal stride
    assert torch.equal(_dense()(odd, k, v), _dense()(odd.contiguous(), k, v))
    one_k, one_v = k[:1].contiguous().requires_grad_(), v[:1].contiguous().requires_grad_()
    out = _dense()(q, one_k.expand(B, -1, -1, -1), one_v.expand(B, -1, -1, -1), causal=True)
    full = [x.detach().repeat(B, 1, 1, 1).requires_grad_() for x in (one_k, one_v)]
    ref = _dense()(q, *full, causal=True)
    assert torch.equal(out, ref)
    dout = torch.randn(out.shape, generator=g, device="cuda").to(out.dtype)
    for a, b in zip(torch.autograd.grad(out, (one_k, one_v), dout), torch.autograd.grad(ref, full, dout)):
        assert torch.equal(a, b.sum(0, keepdim=True))
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    ones = torch.autograd.grad(_dense()(*leaves, causal=True), leaves, torch.ones_like(out))
    for a, b in zip(torch.autograd.grad(_dense()(*leaves, causal=True).sum(), leaves), ones):  # a dout with all strides 0
        assert torch.equal(a, b)


WALKS = {  # with a distance the units of keys come in another order than the keys
    "all_seen": ((1, 3, 1, 700, 700), dict(slopes=True)),
    "more_keys": ((2, 2, 2, 200, 900), dict(slopes=True, cap=30.0)),
    "more_queries": ((1, 2, 1, 900, 200), dict(slopes=True)),  # the first queries stand before the first key
    "prefix_far_ahead": ((1, 2, 2, 600, 600), dict(slopes=True, causal=True, prefix=[[500]])),
    "documents_of_other_lengths": ((1, 2, 2, 500, 640), dict(slopes=True, docs=[([0, 60, 61, 400, 480], [0, 300, 300, 420, 640])])),
    "lengths": ((3, 2, 1, 150, 520), dict(slopes=True, k_lens=[520, 1, 333])),
}


@pytest.mark.parametrize("impl", [TC, MMA])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", WALKS)
def test_walks_with_a_distance(name, D, impl):
    B, Hq, Hk, Sq, Sk = WALKS[name][0]
    lo, hi, pos, kw, scale, _ = _options(WALKS[name], torch.bfloat16, D)
    q, k, v, _ = _inputs(B, Hq, Hk, Sq, Sk, D, torch.bfloat16, seed=11)
    want = R.attend(q, k, v, lo, hi, pos, scale, kw["softcap"], kw["slopes"])
    out, lse = _dense()(q, k, v, return_lse=True, impl=impl, **kw)
    assert R.worst(out, want["o"]) <= 1
    blind = torch.isinf(want["lse"])
    assert torch.equal(torch.isinf(lse), blind) and float((lse.double() - want["lse"])[~blind].abs().max()) <= R.SCORE + 1e-5
    v[:, :, 300 % Sk, 5] = math.inf  # seen by some rows of mixed tiles, by all of whole ones
    lo, hi = (x.to("cuda")[:, None] for x in (lo, hi))
    sees = ((lo <= 300 % Sk) & (hi > 300 % Sk)).expand(B, Hq, Sq)
    out = _dense()(q, k, v, impl=impl, **kw)
    assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 5][~sees]).all() and not torch.isfinite(out[..., 5][sees]).any()


@pytest.mark.parametrize("impl", [TC, MMA])
@pytest.mark.parametrize("cap", [0.0, 400.0])
def test_a_reference_that_moves(impl, cap):
    """Keys from 640 on have scores of four times the size, so that the maximum of most rows jumps there, in whole units and in mixed ones.
    Sums of |q_d k_d| scale stay below 128 * 6 * 4 * 0.64 * 0.02 = 39 on average."""
    q, k, v, _ = _inputs(1, 4, 2, 1100, 1100, 128, torch.bfloat16, seed=12, spread=6.0)
    k[:, :, 640:] *= 4
    lo, hi, pos = R.runs(1, 1100, 1100, True, None, None, None)
    want = R.attend(q, k, v, lo, hi, pos, 0.02, cap)
    out, lse = _dense()(q, k, v, causal=True, scale=0.02, softcap=cap, return_lse=True, impl=impl)
    assert R.worst(out, want["o"]) <= 1 and float((lse.double() - want["lse"]).abs().max()) <= R.SCORE + 1e-5


def _unaligned(t):
    """The same values behind eight bytes of something else, in a storage whose batch stride is odd where there is one batch entry."""
    flat = torch.zeros(2, t.numel() + 9, dtype=t.dtype, device=t.device)
    view = flat[1, 4:4 + t.numel()].view(t.shape)
    if t.shape[0] == 1:
        view = flat.as_strided(t.shape, (t.numel() + 9, *t.stride()[1:]), 8)
    return view.copy_(t)


def test_unaligned_and_single_entry_views():
    for B in (1, 2):
        q, k, v, dout = _inputs(B, 4, 2, 100, 100, 64, torch.float16, seed=8)
        leaves = [x.requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True)
        want = [out, *torch.autograd.grad(out, leaves, dout)]
        odd = [_unaligned(x.detach()).requires_grad_() for x in (q, k, v)]
        assert all(x.is_contiguous() for x in odd)
        out = _dense()(*odd, causal=True)
        assert all(torch.equal(a, b) for a, b in zip(want, [out, *torch.autograd.grad(out, odd, _unaligned(dout))]))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("impl", [TC, MMA])
def test_a_large_cap_keeps_small_scores(impl, D):
    """A cap far above the scores changes nothing, in tiles with scores on its own scale too: the rows whose scores are small keep the bounds
    of every other case (the others' scores are off by 2^-24 of 10^5 and more; their dout is zero)."""
    B, Hq, Hk, S = 1, 4, 2, 150
    q, k, v, dout = _inputs(B, Hq, Hk, S, S, D, torch.bfloat16, seed=9)
    small = torch.arange(S, device="cuda") % 50 != 7
    q = torch.where(small[:, None], q, q * 3e5)
    dout = dout * small[:, None]
    lo, hi, pos = R.runs(B, S, S, True, None, None, None)
    for cap in (80000.0, 2000.0):
        want = R.attend(q, k, v, lo, hi, pos, D ** -0.5, cap, None, dout)
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True, softcap=cap, impl=impl)
        assert R.worst(out[:, :, small], [x[:, :, small] for x in want["o"]]) <= 1
        grads = torch.autograd.grad(out, leaves, dout)
        assert R.worst(grads[0][:, :, small], [x[:, :, small] for x in want["dq"]]) <= 1
        assert R.worst(grads[1], want["dk"]) <= 1 and R.worst(grads[2], want["dv"]) <= 1


@pytest.mark.parametrize("impl", [TC, MMA])
def test_two_calls_give_the_same_bits(impl):
    q, k, v, dout = _inputs(2, 8, 2, 500, 500, 128, torch.bfloat16)
    res = []
    for _ in range(2):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True, softcap=20.0, slopes=_slopes(8), impl=impl)
        res.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_bounds_outside_the_tensors_are_clamped():
    """Documents and lengths that reach beyond the tensors, or begin before them, are cut at their ends."""
    q, k, v, dout = _inputs(1, 2, 2, 100, 100, 64, torch.bfloat16)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    assert torch.equal(_dense()(q, k, v, k_lens=ints(5000)), _dense()(q, k, v))
    assert torch.equal(_dense()(q, k, v, k_lens=ints(-7)), torch.zeros_like(q))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = _dense()(*leaves, cu_q=ints(-50, 200), cu_k=ints(-20, 1 << 30))
    assert torch.equal(out, _dense()(q, k, v))
    assert all(torch.isfinite(x).all() for x in torch.autograd.grad(out, leaves, dout))


def test_empty_tensors():
    q, k, v, _ = _inputs(1, 2, 2, 20, 20, 64, torch.bfloat16)
    out = _dense()(q, k[:, :, :0], v[:, :, :0], causal=True)
    assert torch.equal(out, torch.zeros_like(q))
    assert _dense()(q[:, :, :0], k, v).shape == (1, 2, 0, 64)
    assert _dense()(q[:0], k[:0], v[:0]).shape == (0, 2, 20, 64)
    leaves = [x.requires_grad_() for x in (q.clone(), k[:, :, :0].clone(), v[:, :, :0].clone())]
    grads = torch.autograd.grad(_dense()(*leaves).sum(), leaves)
    assert torch.equal(grads[0], torch.zeros_like(q)) and grads[1].shape == (1, 2, 0, 64)


@pytest.mark.parametrize("Sq,Sk,impl", [(3, 700, MMA), (1, 30000, MMA), (300, 300, TC)])
def test_captured_calls_follow_their_numbers(Sq, Sk, impl):
    """Two graphs of the same call on their own streams: replayed with other lengths, values and slopes."""
    q, k, v, _ = _inputs(2, 4, 2, Sq, Sk, 128, torch.bfloat16)
    lens = torch.tensor([Sk, Sk // 2], dtype=torch.int32, device="cuda")
    slopes = _slopes(4)
    graphs, outs = [], []
    call = lambda: _dense()(q, k, v, causal=True, k_lens=lens, slopes=slopes, softcap=10.0, impl=impl)  # noqa: E731
    call()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    lens.copy_(torch.tensor([Sk // 3, Sk - 1]))
    q.mul_(0.5)
    slopes.mul_(2)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    want = call()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_other_streams():
    """Calls on two streams at once, forward and backward: each has its own workspace."""
    args = [_inputs(1, 16, 8, 700, 700, 64, torch.float16, seed=s) for s in range(2)]

    def step(q, k, v, dout):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True, impl=TC)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    want = [step(*a) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in args], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(*args[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_offsets_beyond_32_bits():
    """A cache whose last entry lies more than 2^32 bytes (and 2^31 elements) behind its first."""
    S, D = 200, 128
    cache = torch.empty(2, 2 ** 30 // D + 64, 2, D, dtype=torch.bfloat16, device="cuda")  # [entry, slot, k or v, D]: 4 GiB each entry
    n = cache.shape[1]
    q = _inputs(2, 4, 1, 1, 1, D, torch.bfloat16)[0]
    cache[:, n - S:] = torch.randn(2, S, 2, D, device="cuda").to(torch.bfloat16)
    k, v = cache[:, :, 0][:, None], cache[:, :, 1][:, None]
    cu_q, cu_k = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([n - S, n], dtype=torch.int32, device="cuda")
    out = _dense()(q, k, v, cu_q=cu_q, cu_k=cu_k)
    assert torch.isfinite(out).all()
    near = _dense()(q, k[:, :, n - S:], v[:, :, n - S:])
    assert R.worst(out, R.attend(q, k[:, :, n - S:], v[:, :, n - S:], *R.runs(2, 1, S, False, None, None, None), 1 / math.sqrt(D))["o"]) <= 1
    assert float((out.double() - near.double()).abs().max()) < 0.05


def test_refusals_on_the_gpu():
    q, k, v, _ = _inputs(1, 4, 2, 8, 8, 64, torch.bfloat16)
    dense = _dense()
    from longcat_video_b200._lib import LcbsaError
    for bad in (lambda: dense(q[..., :32], k[..., :32], v[..., :32]), lambda: dense(q[:, :3], k, v), lambda: dense(q, k, v[:, :, :4]),
                lambda: dense(q.float(), k.float(), v.float())):
        with pytest.raises(LcbsaError):
            bad()
    with pytest.raises(ValueError):
        dense(q, k.half(), v.half())
    with pytest.raises(TypeError):
        dense(q.double(), k.double(), v.double())
    with pytest.raises(TypeError):
        dense(q, k, v, k_lens=torch.ones(1, device="cuda"))
    with pytest.raises(ValueError):
        dense(q, k, v, k_lens=torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        dense(q, k, v, slopes=torch.ones(4, device="cuda", requires_grad=True))


def test_no_second_derivative():
    """A gradient that is itself differentiated says so instead of coming out as zero."""
    from longcat_video_b200.modules import embed_rotary, rotary_frequencies
    q, k, v, dout = _inputs(1, 2, 2, 70, 70, 64, torch.bfloat16)
    q.requires_grad_()
    for out in (_dense()(q, k, v), embed_rotary(q, rotary_frequencies(64))):
        (dq,) = torch.autograd.grad(out, q, dout.requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            dq.sum().backward()


def test_versions_of_saved_tensors_are_checked():
    q, k, v, dout = _inputs(1, 2, 2, 70, 70, 64, torch.bfloat16)
    leaf = q.clone().requires_grad_()
    k = k.clone()
    out = _dense()(leaf, k, v)
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward(dout)


@pytest.mark.parametrize("D,dtype,kw", [(128, torch.bfloat16, dict(causal=True)), (64, torch.float16, dict(softcap=8.0, slopes=True)),
                                        (64, torch.bfloat16, dict(causal=True, docs=True))])
def test_many_items_per_cta(D, dtype, kw):
    """More tiles than SMs, several to a CTA, of very different lengths: every head gives the bits it gives alone, and a few of
    them are held to the formulas."""
    B, Hq, Hk, S = 3, 40, 40, 700
    kw = dict(kw)
    if kw.pop("docs", False):
        kw["cu_q"] = torch.tensor([[0, 90, 91, 600, 700], [0, 0, 300, 300, 700], [5, 100, 200, 500, 650]], dtype=torch.int32, device="cuda")
    slopes = _slopes(Hq) if kw.pop("slopes", False) else None
    q, k, v, dout = _inputs(B, Hq, Hk, S, S, D, dtype, seed=7)

    def step(q, k, v, dout, slopes):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, slopes=slopes, impl=TC, **kw)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    full = step(q, k, v, dout, slopes)
    for h in (0, 17, 39):
        one = step(*(x[:, h:h + 1] for x in (q, k, v, dout)), None if slopes is None else slopes[h:h + 1])
        for a, b in zip(full, one):
            assert torch.equal(a[:, h:h + 1], b)
    docs = None if "cu_q" not in kw else [(c, c) for c in kw["cu_q"].tolist()]
    lo, hi, pos = R.runs(B, S, S, kw.get("causal", False), docs, None, None)
    want = R.attend(*(x[:, 17:19] for x in (q, k, v)), lo, hi, pos, 1 / math.sqrt(D), kw.get("softcap", 0.0), None if slopes is None else slopes[17:19],
                    dout[:, 17:19])
    for got, x in zip(full, ("o", "dq", "dk", "dv")):
        assert R.worst(got[:, 17:19], want[x]) <= 1, x


def test_waves_of_heads():
    """K and V of all heads together exceed what the items' order keeps in the L2: heads in waves, each with the bits it has alone."""
    H, S, D = 37, 4096, 128
    q, k, v, dout = _inputs(1, H, H, S, S, D, torch.bfloat16)

    def step(q, k, v, dout):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True, impl=TC)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    full = step(q, k, v, dout)
    for h in (0, 18, 19, 36):
        for a, b in zip(full, step(*(x[:, h:h + 1] for x in (q, k, v, dout)))):
            assert torch.equal(a[:, h:h + 1], b)


@pytest.mark.parametrize("B,Hq,Hk,Sq,Sk,D", [(1, 4, 1, 1, 20000, 128), (1, 2, 1, 3, 12345, 64), (40, 8, 4, 1, 2100, 128), (2, 16, 2, 3, 900, 64),
                                             (1, 1, 1, 1, 65, 128), (70, 4, 4, 2, 130, 64), (1, 64, 2, 1, 515, 128)])
def test_ways_of_sharing_out_the_keys(B, Hq, Hk, Sq, Sk, D):
    """Chunks with a second kernel, clusters of every size, one CTA; one tile of rows and several of two."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, Sk + 1, (B,), generator=g).tolist()
    lens[0] = Sk
    q, k, v, _ = _inputs(B, Hq, Hk, Sq, Sk, D, torch.bfloat16)
    lo, hi, pos = R.runs(B, Sq, Sk, True, None, lens, None)
    want = R.attend(q, k, v, lo, hi, pos, 1 / math.sqrt(D), 25.0, _slopes(Hq))
    out, lse = _dense()(q, k, v, causal=True, softcap=25.0, slopes=_slopes(Hq), k_lens=torch.tensor(lens, device="cuda"), return_lse=True, impl=MMA)
    assert R.worst(out, want["o"]) <= 1
    blind = torch.isinf(want["lse"])
    assert torch.equal(torch.isinf(lse), blind) and float((lse.double() - want["lse"])[~blind].abs().max()) <= R.SCORE + 1e-5


def test_scores_of_any_size_under_a_cap():
    """Scores far beyond the cap, where the polynomial does not reach, next to small ones."""
    for impl in (TC, MMA):
        q, k, v, dout = _inputs(1, 2, 2, 200, 200, 64, torch.bfloat16, seed=9)
        q[:, :, 30:40] *= 40
        lo, hi, pos = R.runs(1, 200, 200, True, None, None, None)
        want = R.attend(q, k, v, lo, hi, pos, 0.02, 2.0, None, dout)
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, causal=True, softcap=2.0, scale=0.02, impl=impl)
        assert R.worst(out.detach(), want["o"]) <= 1
        for got, x in zip(torch.autograd.grad(out, leaves, dout), ("dq", "dk", "dv")):
            assert R.worst(got, want[x]) <= 1, x


def test_a_scale_of_zero():
    q, k, v, dout = _inputs(1, 2, 2, 150, 150, 64, torch.bfloat16)
    for impl in (TC, MMA):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = _dense()(*leaves, scale=0.0, softcap=3.0, impl=impl)
        mean = v.double().mean(2, keepdim=True)
        assert float((out.detach().double() - mean).abs().max()) <= 2.0 ** -8 * 2 * float(v.detach().abs().max())
        dq, dk, dv = torch.autograd.grad(out, leaves, dout)
        assert not dq.any() and not dk.any() and torch.isfinite(dv).all()


def test_a_step_in_a_graph_beside_an_eager_one():
    """Forward and gradients captured while an eager graph of the same leaves lives: refused at the call, before the capture breaks
    in the engine.  With the eager graph released the same capture goes through and gives the same."""
    q, k, v, dout = _inputs(1, 4, 2, 300, 300, 64, torch.bfloat16)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    call = lambda: _dense()(*leaves, causal=True, softcap=9.0)  # noqa: E731
    eager = call()
    with pytest.raises(RuntimeError, match="live graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    want = [eager.detach(), *torch.autograd.grad(eager, leaves, dout)]
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
        grads = torch.autograd.grad(out, leaves, dout)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((out, *grads), want))
