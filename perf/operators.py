"""The work the dense attention and the 1-D rotary embedding of this library are measured on.

Both stand beside the block-sparse attention of the video DiT: its text encoder, its cross-attention to packed prompts, its
layers without block sparsity and an autoregressive model that shares the GPU call ``dense_attention`` and
``embed_rotary_qk`` of ``longcat_video_b200.modules``.  A case is a dict of plain values:

  op        "attend": the attention alone   "train": the attention and its gradients
            "rotary": q and k embedded      "rotary_train": the same and the gradients
  batch, heads, kv_heads, head_dim, dtype   heads / kv_heads query heads share a key head
  q_len, k_len  tokens of q and of k, v     (rotary: q_len tokens of both)
  docs      documents packed behind each other in every batch entry (0: the whole sequence is one)
  ragged    with docs 0: the keys behind a length of the batch entry's own are not looked at (a padded cache)
  causal    a query sees no key behind its own position; the last query of a document stands at its last key
  prefix    that many first keys of a document are seen by all its queries (with causal)
  cap       scores s become cap * tanh(s / cap); 0: as they are
  slopes    the distance |position - key| times a slope of the head is taken off the score
  rotary_dim, interleaved, base, scaling    first dimensions of the head that turn; pairs (2i, 2i+1) or (i, i + rotary_dim/2)
  far       the positions reach up to this one
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _attend(op, batch, heads, kv_heads, q_len, k_len, head_dim=128, dtype="bf16", docs=0, ragged=False, causal=True, prefix=0, cap=0.0,
            slopes=False):
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len, "k_len": k_len, "head_dim": head_dim, "dtype": dtype,
            "docs": docs, "ragged": ragged, "causal": causal, "prefix": prefix, "cap": cap, "slopes": slopes}


def _rotary(op, batch, heads, kv_heads, q_len, head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16", base=10000.0, scaling="none", far=0):
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len, "head_dim": head_dim, "rotary_dim": rotary_dim,
            "interleaved": interleaved, "dtype": dtype, "base": base, "scaling": scaling, "far": far}


def listed():
    cases = {
        # one token of one sequence behind a short cache: latency is what counts
        "token_short": _attend("attend", 1, 32, 8, 1, 1023, cap=30.0),
        # one token of each of 32 sequences behind caches of up to 32768 keys, ragged: the cache is read once
        "token_cache": _attend("attend", 32, 32, 8, 1, 32768, ragged=True, slopes=True),
        # five drafted tokens each of eight sequences, a small fp16 model
        "draft_tokens": _attend("attend", 8, 16, 4, 5, 9001, head_dim=64, dtype="fp16", ragged=True),
        # a text encoder on a short padded prompt: bidirectional, biased by distance
        "encode_prompt": _attend("attend", 2, 12, 12, 197, 197, head_dim=64, dtype="fp16", ragged=True, causal=False, slopes=True),
        # several prompts packed into one row and read at once, capped scores
        "packed_prompts": _attend("attend", 1, 16, 4, 9973, 9973, docs=7, cap=50.0),
        # the DiT's cross-attention: the video tokens of two samples, each against its own text
        "video_to_text": _attend("attend", 1, 32, 32, 9984, 1024, docs=2, causal=False),
        # a training step of a small fp16 model with a bidirectional prefix
        "train_small": _attend("train", 2, 8, 8, 511, 511, head_dim=64, dtype="fp16", prefix=100, slopes=True),
        # a training step on packed documents, capped scores
        "train_packed": _attend("train", 1, 16, 4, 5000, 5000, docs=9, cap=30.0),
        # a training step on one long document with a prefix and distances: the largest product
        "train_long": _attend("train", 1, 16, 8, 8192, 8192, prefix=1000, slopes=True),
        # q and k of one token of each of 16 sequences far into a long context
        "rotary_token": _rotary("rotary", 16, 32, 8, 1, scaling="parts", base=500000.0, far=1000000),
        # q and k of a prompt, half of the head, pairs next to each other
        "rotary_prompt": _rotary("rotary", 1, 16, 4, 5003, rotary_dim=64, interleaved=True, dtype="fp16", scaling="linear"),
        # q and k of a training batch and their gradients
        "rotary_step": _rotary("rotary_train", 2, 32, 32, 8192),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 6, 8])
    d, t = rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    shape = dict(head_dim=d, dtype=t, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.4)
    kind = rng.choice(["token", "attend", "cross", "train", "train", "rotary"])
    if kind == "token":
        k = log(64, 32768)
        return _attend("attend", max(1, min(rng.randint(1, 32), 4000000 // (k * kv))), kv * group, kv, rng.choice([1, 1, 1, 2, 3, 4, 7, 8]), k,
                       ragged=rng.random() < 0.7, causal=rng.random() < 0.8, **shape)
    if kind == "rotary":
        r = rng.choice([16 * i for i in range(1, d // 16 + 1)])
        op, n = rng.choice(["rotary", "rotary_train"]), log(1, 16384)
        return _rotary(op, max(1, min(rng.randint(1, 8), 16384 // n)), kv * group, kv, n, d, r, rng.random() < 0.5, t, rng.choice([10000.0, 500000.0]),
                       rng.choice(["none", "linear", "base", "parts", "wave"]), rng.choice([0, 100000, 1000000]))
    n = log(100, 8192 if kind != "train" else 6000)
    b = max(1, min(rng.randint(1, 4), 9000 // n))
    heads = kv * group
    while heads > kv and b * heads * n * n > 900000000:
        heads -= kv
    kv = min(kv, heads)
    if b * heads * n * n > 900000000:
        heads = kv = max(1, 900000000 // (b * n * n))
    if kind == "cross":
        return _attend("attend", b, heads, kv, n, log(20, 1024), docs=rng.randint(1, 6), causal=False, **shape)
    causal = rng.random() < 0.75
    docs = rng.choice([0, 0, 1, 3, 8, 20])
    return _attend("train" if kind == "train" else "attend", b, heads, kv, n, n, docs=docs, ragged=docs == 0 and rng.random() < 0.3, causal=causal,
                   prefix=rng.choice([0, 0, n // 5]) if causal else 0, **shape)


# --------------------------------------------------------------------------------------------------------- the inputs


def _bounds(case):
    """Where the documents of each batch entry begin in q and in k, [batch][docs + 1], or the lengths of its keys: a
    function of the case alone."""
    rng = random.Random(case["q_len"] * 7919 + case["k_len"] * 31 + case["docs"])
    if case["docs"]:
        rows = []
        for _ in range(case["batch"]):
            cuts = sorted(rng.random() for _ in range(case["docs"] - 1))
            rows.append([[0] + [int(c * n) for c in cuts] + [n] for n in (case["q_len"], case["k_len"])])
        return [r[0] for r in rows], [r[1] for r in rows]
    lens = [rng.randint(max(1, case["k_len"] // 4), case["k_len"]) if case["ragged"] else case["k_len"] for _ in range(case["batch"])]
    return [[0, case["q_len"]]] * case["batch"], [[0, n] for n in lens]


def _pairs(case):
    """Pairs of a query and a key that it sees, over the batch, and the keys that are seen at all."""
    pairs = keys = 0
    for cu_q, cu_k in zip(*_bounds(case)):
        for q0, q1, k0, k1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
            n, m = q1 - q0, k1 - k0
            keys += m
            if not case["causal"]:
                pairs += n * m
                continue
            p = min(case["prefix"], m)
            pairs += sum(max(p, min(m, max(0, m - n + 1 + i))) for i in range(n))
    return pairs, keys


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, b, hq, hk, d, n = _DTYPES[case["dtype"]], case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["q_len"]
    new = lambda *size: torch.randn(*size, generator=gen, device="cuda", dtype=t)  # noqa: E731
    state = {"case": dict(case)}
    if case["op"].startswith("rotary"):
        qkv = new(b, n, hq + 2 * hk, d)  # the fused projection of a layer: q and k are views of it
        state["q"], state["k"] = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hk].transpose(1, 2)
        last = torch.randint(n, max(case["far"], n) + 1, (b, 1), generator=gen, device="cuda")
        state["positions"] = last - n + torch.arange(n, device="cuda")
        if case["op"] == "rotary_train":
            state["dq"], state["dk"] = new(b, hq, n, d), new(b, hk, n, d)
        return state
    m = case["k_len"]
    if n == m:
        qkv = new(b, n, hq + 2 * hk, d)
        q, k, v = (x.transpose(1, 2) for x in qkv.split([hq, hk, hk], dim=2))
    else:
        q, k, v = new(b, n, hq, d).transpose(1, 2), new(b, hk, m, d), new(b, hk, m, d)
    state["q"], state["k"], state["v"] = q, k, v
    if case["op"] == "train":
        state["dout"] = new(b, hq, n, d)
    if case["slopes"]:
        state["slopes"] = 0.5 ** (1 + torch.arange(hq, device="cuda", dtype=torch.float32) * 8 / hq)
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in _bounds(case))
    if case["docs"]:
        state["cu_q"], state["cu_k"] = cu_q, cu_k
    elif case["ragged"]:
        state["k_lens"] = cu_k[:, 1].contiguous()
    if case["prefix"]:
        state["prefix"] = torch.full((b, max(1, case["docs"])), case["prefix"], dtype=torch.int32, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------------ the plain form


def _inv_freq(case):
    """Radians per position of the pairs, in 64 bits, after the scaling for long contexts, and the factor on the result."""
    r, base, factor = case["rotary_dim"], case["base"], 1.0
    if case["scaling"] == "base":
        base = base * 4.0 ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    if case["scaling"] == "linear":
        f = f / 4
    elif case["scaling"] == "parts":  # pairs that turn more than 32 times within 8192 positions stay, those below one turn are slowed
        at = lambda turns: r * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), r - 1)
        ramp = ((torch.arange(r // 2, device="cuda", dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / 16 * ramp + f * (1 - ramp)
        factor = 0.1 * math.log(16) + 1
    elif case["scaling"] == "wave":  # by wavelength: above 8192 slowed, below 8192 / 4 as they are
        smooth = ((8192 * f / (2 * math.pi) - 1) / 3).clamp(0, 1)
        f = f / 8 * (1 - smooth) + f * smooth
    return f, factor


_SCALING = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "base": {"kind": "base", "factor": 4.0},
            "parts": {"kind": "by_parts", "factor": 16.0, "original_length": 8192},
            "wave": {"kind": "by_wavelength", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 4.0}}


def _turn(x, cos, sin, r, interleaved):
    head, rest = x[..., :r], x[..., r:]
    a, b = (head[..., ::2], head[..., 1::2]) if interleaved else (head[..., : r // 2], head[..., r // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([head, rest], dim=-1)


def _rotary_plain(s):
    case = s["case"]
    inv, factor = _inv_freq(case)
    angle = s["positions"][:, None, :, None].double() * inv  # far positions: the angle needs more than 24 bits
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    r, inter = case["rotary_dim"], case["interleaved"]
    if case["op"] == "rotary":
        return [_turn(s[x].float(), cos, sin, r, inter).to(s[x].dtype) for x in ("q", "k")]
    out = [_turn(s[x].float(), cos, sin, r, inter).to(s[x].dtype) for x in ("q", "k")]
    return out + [_turn(s[x].float(), cos, -sin, r, inter).to(s[x].dtype) for x in ("dq", "dk")]


def _seen(s, device="cuda"):
    """[batch, q_len, k_len] whether a query sees a key, and [batch, q_len] the position of a query among the keys."""
    case = s["case"]
    i = torch.arange(case["q_len"], device=device).expand(case["batch"], -1).contiguous()
    j = torch.arange(case["k_len"], device=device).expand(case["batch"], -1).contiguous()
    if case["docs"]:
        cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    else:
        cu_k = torch.full((case["batch"], 2), case["k_len"], device=device)
        cu_k[:, 0] = 0
        if case["ragged"]:
            cu_k[:, 1] = s["k_lens"]
        cu_q = torch.tensor([[0, case["q_len"]]], device=device).expand(case["batch"], -1).contiguous()
    doc_i, doc_j = (torch.searchsorted(cu, x, right=True) - 1 for cu, x in ((cu_q, i), (cu_k, j)))
    doc_j = torch.where(j < cu_k[:, -1:], doc_j, -1)
    end = lambda cu, doc: cu.gather(1, (doc + 1).clamp(max=cu.shape[1] - 1))  # noqa: E731
    pos = end(cu_k, doc_i) - (end(cu_q, doc_i) - i)
    seen = doc_i[:, :, None] == doc_j[:, None, :]
    if case["causal"]:
        early = j[:, None, :] <= pos[:, :, None]
        if case["prefix"]:
            early = early | ((j - cu_k.gather(1, doc_j.clamp(min=0))) < case["prefix"])[:, None, :]
        seen = seen & early
    return seen, pos


def _attend_plain(s, q, k, v):
    """softmax over the seen keys of cap * tanh(q k / sqrt(d) / cap) - slope * distance, times v; rows that see nothing are 0."""
    case = s["case"]
    seen, pos = _seen(s)
    b, hq, n, d = q.shape
    hk, m = k.shape[1], k.shape[2]
    x = (q.reshape(b, hk, -1, d) @ k.transpose(-1, -2)).view(b, hq, n, m) * (1 / math.sqrt(d))
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    if case["slopes"]:
        away = (pos[:, :, None] - torch.arange(m, device="cuda")).abs().float()
        x = x - s["slopes"][:, None, None] * away[:, None]
    x = x.masked_fill(~seen[:, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).detach().clamp(min=-1e30))
    p = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    return (p.view(b, hk, -1, m) @ v).view(b, hq, n, d)


def _options(s):
    case = s["case"]
    return dict(causal=case["causal"], softcap=case["cap"], slopes=s.get("slopes"), cu_q=s.get("cu_q"), cu_k=s.get("cu_k"), k_lens=s.get("k_lens"),
                prefix_lens=s.get("prefix"))


def run(state):
    case, s = state["case"], state
    if case["op"].startswith("rotary"):
        if not own:
            return _rotary_plain(s)
        from longcat_video_b200.modules import embed_rotary_qk, rotary_frequencies
        freqs = rotary_frequencies(case["rotary_dim"], case["base"], _SCALING[case["scaling"]])
        if case["op"] == "rotary":
            return list(embed_rotary_qk(s["q"], s["k"], freqs, s["positions"], interleaved=case["interleaved"]))
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        out = embed_rotary_qk(q, k, freqs, s["positions"], interleaved=case["interleaved"])
        return [x.detach() for x in out] + list(torch.autograd.grad(out, (q, k), (s["dq"], s["dk"])))
    t = s["q"].dtype
    if case["op"] == "attend":
        if own:
            from longcat_video_b200.modules import dense_attention
            return dense_attention(s["q"], s["k"], s["v"], **_options(s))
        return _attend_plain(s, s["q"].float(), s["k"].float(), s["v"].float()).to(t)
    if own:
        from longcat_video_b200.modules import dense_attention
        q, k, v = (s[x].detach().requires_grad_() for x in ("q", "k", "v"))
        out = dense_attention(q, k, v, **_options(s))
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), s["dout"])]
    q, k, v = (s[x].detach().float().requires_grad_() for x in ("q", "k", "v"))
    out = _attend_plain(s, q, k, v)
    return [x.detach().to(t) for x in (out, *torch.autograd.grad(out, (q, k, v), s["dout"].float()))]


def work(case):
    d, e = case["head_dim"], 2
    b, hq, hk, n = case["batch"], case["heads"], case["kv_heads"], case["q_len"]
    if case["op"].startswith("rotary"):
        passes = 2 if case["op"] == "rotary" else 4  # q and k in and out; the gradients in and out
        return {"bytes": passes * b * n * (hq + hk) * d * e + 8 * b * n, "flops": passes // 2 * 3 * b * n * (hq + hk) * case["rotary_dim"]}
    pairs, keys = _pairs(case)
    q, kv = b * hq * n * d * e, hk * keys * d * e
    if case["op"] == "attend":
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * hq * d}
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * hq * d}  # q, dout in, out, dq out; k, v in, dk, dv out; two products there, five back


# ------------------------------------------------------------------------------------------------------- in 64 bits


def _exact_rotary(s):
    """Every pair as a complex number times exp(i angle), the angle reduced in turns."""
    case = s["case"]
    inv, factor = _inv_freq(case)
    turns = s["positions"][:, None, :, None].double() * (inv / (2 * math.pi))
    turns = turns - turns.round()
    turn = torch.polar(torch.full_like(turns, factor), turns * (2 * math.pi))
    r, h = case["rotary_dim"], case["rotary_dim"] // 2
    out = []
    for name in ("q", "k") if case["op"] == "rotary" else ("q", "k", "dq", "dk"):
        x = s[name].double()
        t = turn.conj() if name[0] == "d" else turn
        y = x.clone()
        if case["interleaved"]:
            z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * t
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :h], x[..., h:r]) * t
            y[..., :h], y[..., h:r] = z.real, z.imag
        out.append(y)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("rotary"):
        return _exact_rotary(s)
    b, hq, hk, d, n, m = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim", "q_len", "k_len"))
    out = torch.zeros(b, hq, n, d, device="cuda", dtype=torch.float64)
    grads = [torch.zeros(b, h, x, d, device="cuda", dtype=torch.float64) for h, x in ((hq, n), (hk, m), (hk, m))]
    for e, (cu_q, cu_k) in enumerate(zip(*_bounds(case))):
        for q0, q1, k0, k1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
            if q1 == q0 or k1 == k0:
                continue
            i, j = torch.arange(q0, q1, device="cuda")[:, None], torch.arange(k0, k1, device="cuda")[None, :]
            away = (k1 - q1 + i) - j
            hidden = (away < 0) & (j - k0 >= case["prefix"]) if case["causal"] else torch.zeros_like(away, dtype=torch.bool)
            for h in range(hq):
                g = h // (hq // hk)
                q, k, v = s["q"][e, h, q0:q1].double(), s["k"][e, g, k0:k1].double(), s["v"][e, g, k0:k1].double()
                x = torch.mm(q, k.t()) / d ** 0.5
                if case["cap"]:
                    x = torch.tanh(x / case["cap"])
                    slack = 1 - x * x
                    x = x * case["cap"]
                if case["slopes"]:
                    x = x - s["slopes"][h].double() * away.abs()
                x[hidden] = -math.inf
                blind = hidden.all(1)
                p = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
                p[blind] = 0
                out[e, h, q0:q1] = o = torch.mm(p, v)
                if case["op"] == "train":
                    do = s["dout"][e, h, q0:q1].double()
                    ds = p * (torch.mm(do, v.t()) - (do * o).sum(1, keepdim=True)) / d ** 0.5
                    if case["cap"]:
                        ds = ds * slack
                    grads[0][e, h, q0:q1] = torch.mm(ds, k)
                    grads[1][e, g, k0:k1] += torch.mm(ds.t(), q)
                    grads[2][e, g, k0:k1] += torch.mm(p.t(), do)
    return out if case["op"] == "attend" else [out, *grads]
