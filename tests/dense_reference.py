"""The dense attention and the 1-D rotary embedding written out in 64 bits, and how far a kernel may be from them.

``attend`` also returns elementwise bounds, from the roundings a kernel that keeps its sums in fp32 makes; u is half a step of the
input type relative to a value (2^-8 bf16, 2^-11 fp16), t half its smallest step (fp16: 2^-25):

  scores     fp32 sum of D products, the cap and the distance: together at most SCORE absolute for the inputs of these tests, whose
             sums of |q_d k_d| scale stay below 40: 128 * 2^-24 * 40 = 3.1e-4 in the worst order
  o          P rounded to the type: u |p| + t;  p itself: 2 SCORE (its score and the row's log-sum-exp);  the result: u |o|
  dv         the same with dout in the place of v, summed over queries and heads
  dq, dk     dS rounded: u |ds| + t;  delta from the rounded o: sum_d |dout_d| u |o_d|;  p: 2 SCORE;  the result: u |dq|
"""
import math
from fractions import Fraction

import torch

SCORE = 3.2e-4


def runs(B, Sq, Sk, causal, docs, k_lens, prefix):
    """lo, hi, pos of every query, [B, Sq] each, by loops.  docs: per entry (cu_q, cu_k) lists, or None."""
    lo, hi, pos = (torch.zeros(B, Sq, dtype=torch.int64) for _ in range(3))
    for b in range(B):
        cu_q, cu_k = docs[b] if docs is not None else ([0, Sq], [0, Sk if k_lens is None else k_lens[b]])
        for d in range(len(cu_q) - 1):
            k0, k1 = cu_k[d], cu_k[d + 1]
            for i in range(max(cu_q[d], 0), min(cu_q[d + 1], Sq)):
                p = k1 - (cu_q[d + 1] - i)
                end = k1 if not causal else min(max(p + 1, k0 + (prefix[b][d] if prefix is not None else 0), k0), k1)
                lo[b, i], hi[b, i], pos[b, i] = k0, end, p
    return lo, hi, pos


def attend(q, k, v, lo, hi, pos, scale, cap=0.0, slopes=None, dout=None):
    """Returns a dict of (value, bound) for o and, with dout, dq, dk, dv; and lse."""
    dev, t = q.device, q.dtype
    u = torch.finfo(t).eps / 2
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    B, Hq, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    G = Hq // Hk
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    lo, hi, pos = (x.to(dev)[:, None, :, None] for x in (lo, hi, pos))
    j = torch.arange(Sk, device=dev)
    seen = (j >= lo) & (j < hi)
    s = q @ k.transpose(-1, -2) * scale
    slack = torch.ones_like(s)
    if cap:
        th = torch.tanh(s / cap)
        s, slack = cap * th, 1 - th * th
    if slopes is not None:
        s = s - slopes.double()[None, :, None, None] * (pos - j).abs()
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    blind = ~seen.any(-1).expand(B, Hq, Sq)
    p = torch.exp(s - lse.masked_fill(blind, 0.0)[..., None])
    clean = lambda x, m: torch.where(m, x, torch.zeros((), dtype=x.dtype, device=dev))  # noqa: E731
    vz = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
    o = p @ vz
    spread = (u + 2 * SCORE) * (p @ vz.abs()) + tiny * (seen.double() @ vz.abs())
    res = {"o": (o, spread + u * o.abs() + tiny), "lse": lse}
    if dout is None:
        return res
    g = dout.double()
    dp = g @ v.transpose(-1, -2)
    delta = (g * o).sum(-1, keepdim=True)
    d_delta = (g.abs() * (res["o"][1])).sum(-1, keepdim=True)
    ds = p * (dp - delta) * slack * scale
    d_ds = u * ds.abs() + tiny * seen + p * slack * abs(scale) * (d_delta + 2 * SCORE * (dp.abs() + delta.abs()))
    d_ds = d_ds + p * abs(scale) * (dp - delta).abs() * (2 * SCORE if cap else 0.0)  # 1 - tanh^2 from the rounded score
    ds, d_ds = clean(ds, seen), clean(d_ds, seen)
    dq = ds @ k
    fold = lambda x: x.view(B, Hk, G, Sk, D).sum(2)  # noqa: E731
    dk, dv = fold(ds.transpose(-1, -2) @ q), fold(p.transpose(-1, -2) @ g)
    res["dq"] = (dq, d_ds @ k.abs() + u * dq.abs() + tiny)
    res["dk"] = (dk, fold(d_ds.transpose(-1, -2) @ q.abs()) + u * dk.abs() + tiny)
    res["dv"] = (dv, fold(((u + 2 * SCORE) * p + tiny * seen).transpose(-1, -2) @ g.abs()) + u * dv.abs() + tiny)
    return res


def worst(got, value_and_bound):
    """The largest error in units of its bound."""
    value, bound = value_and_bound
    err = (got.double() - value).abs()
    assert torch.isfinite(got.double()).all()
    return float((err / (bound + 1e-9)).detach().max()) if err.numel() else 0.0


def rotate(x, radians, factor, positions, interleaved, inverse=False):
    """positions [B, S]; complex products in 64 bits.  The turns are exact fractions: position * frequency in doubles is off by
    2^-53 of its size, which at position 2^40 is 10^-4 radians."""
    r = 2 * len(radians)
    pi = Fraction("3.14159265358979323846264338327950288419716939937510")
    per = [round(Fraction(f) / (2 * pi) * 2 ** 128) for f in radians]  # turns per position in units of 2^-128
    frac = {}
    for p in set(positions.flatten().tolist()):
        frac[p] = [float(Fraction((p * t) % 2 ** 128, 2 ** 128)) for t in per]
    turns = torch.tensor([[frac[p] for p in row] for row in positions.tolist()], dtype=torch.float64, device=x.device)[:, None]
    z = torch.polar(torch.full_like(turns, factor), turns * (2 * math.pi) * (-1 if inverse else 1))
    x = x.double()
    y = x.clone()
    if interleaved:
        w = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * z
        y[..., 0:r:2], y[..., 1:r:2] = w.real, w.imag
    else:
        w = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * z
        y[..., :r // 2], y[..., r // 2:r] = w.real, w.imag
    return y
