"""Dense attention with capped or distance-biased scores and document, prefix and length masks.

What stands beside the block-sparse attention of the DiT: its cross-attention from the video tokens to packed prompts
(``MultiHeadCrossAttention`` with ``kv_seqlen``, longcat_video/modules/attention.py:184-260, a document mask), its
self-attention with block sparsity off (attention.py:67-104), a text encoder whose scores are biased by distance, an
autoregressive model that shares the GPU.  Forward, backward, and a form for a few tokens of every sequence behind a long cache.
All arithmetic is in liblcbsa.so (``lcbsa_dense_attn_fwd`` / ``_bwd``); there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _lib as L

_PACK_SCORES = struct.Struct("@ff5P2q2i").pack  # the layout of LcbsaScores
assert struct.calcsize("@ff5P2q2i") == ctypes.sizeof(L.LcbsaScores)


class _Shape(NamedTuple):
    """The scores as ``LcbsaScores`` has them; the tensors are kept so that they outlive the launch (and the backward's)."""
    scale: float
    cap: float
    causal: bool
    slopes: Optional[torch.Tensor]
    cu_q: Optional[torch.Tensor]
    cu_k: Optional[torch.Tensor]
    k_lens: Optional[torch.Tensor]
    prefix: Optional[torch.Tensor]

    def packed(self) -> bytes:
        at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        docs = cu_stride = prefix_stride = 0
        if self.cu_q is not None:
            docs = self.cu_q.shape[-1] - 1
            cu_stride = docs + 1 if self.cu_q.dim() == 2 else 0
        if self.prefix is not None and self.prefix.dim() == 2:
            prefix_stride = self.prefix.shape[-1]
        return _PACK_SCORES(self.scale, self.cap, at(self.slopes), at(self.cu_q), at(self.cu_k), at(self.k_lens), at(self.prefix), cu_stride,
                            prefix_stride, docs, self.causal)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B: int, Hq: int, Hk: int, Sq: int, Sk: int, D: int, backward: int) -> int:
    """A pure function of the sizes, asked of the library once."""
    sizes = [L.LcbsaTensor(None, L.LCBSA_BF16, 0, (ctypes.c_int64 * 4)(B, h, n, D)) for h, n in ((Hq, Sq), (Hk, Sk))]
    return L.lib().lcbsa_dense_attn_workspace_bytes(ctypes.byref(sizes[0]), ctypes.byref(sizes[1]), backward)


def _numbers(name: str, t: torch.Tensor, device, shapes) -> torch.Tensor:
    """An int32 tensor of one of the shapes on the call's device, contiguous."""
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, q on {device}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {' or '.join(map(str, shapes))}")
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _shape_of(q, k, causal, softcap, slopes, cu_q, cu_k, k_lens, prefix_lens, scale) -> _Shape:
    B, Hq, _, D = q.shape
    dev = q.device
    softcap = float(softcap)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not math.isfinite(softcap) or softcap < 0:
        raise ValueError(f"softcap {softcap}: 0 (none) or a positive number")
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale} is not finite")
    docs = 1
    if cu_q is not None or cu_k is not None:
        if cu_q is None:
            raise ValueError("cu_k needs cu_q: the documents of the queries")
        if k_lens is not None:
            raise ValueError("cu_q and k_lens exclude each other")
        if cu_k is None:
            cu_k = cu_q
        if cu_q.dim() not in (1, 2) or cu_q.shape[-1] < 2:
            raise ValueError("cu_q must be [docs + 1] or [batch, docs + 1] with at least one document")
        docs = cu_q.shape[-1] - 1
        shapes = ((docs + 1,),) if cu_q.dim() == 1 else ((B, docs + 1),)
        cu_q, cu_k = _numbers("cu_q", cu_q, dev, shapes), _numbers("cu_k", cu_k, dev, shapes)
    elif k_lens is not None:
        k_lens = _numbers("k_lens", k_lens, dev, ((B,),))
    if prefix_lens is not None:
        if not causal:
            raise ValueError("prefix_lens needs causal=True: without it every query sees the whole document")
        prefix_lens = _numbers("prefix_lens", prefix_lens, dev, ((docs,), (B, docs)))
    if slopes is not None:
        if tuple(slopes.shape) != (Hq,):
            raise ValueError(f"slopes has shape {tuple(slopes.shape)}, expected {(Hq,)}")
        if slopes.device != dev:
            raise ValueError(f"slopes is on {slopes.device}, q on {dev}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise ValueError("slopes are constants: they have no gradient")
        slopes = slopes.detach().to(torch.float32).contiguous()
    return _Shape(scale, softcap, bool(causal), slopes, cu_q, cu_k, k_lens, prefix_lens)


_DENSE = torch.contiguous_format


def _forward(q, k, v, shape: _Shape, need_lse: bool, need_rest: bool = False):
    dev = q.device
    out = torch.empty_like(q, memory_format=_DENSE)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev) if need_lse else None
    rest = torch.empty_like(out) if need_rest else None
    (q, qd), (k, kd), (v, vd), (_, od) = L.packed_rows(q), L.packed_rows(k), L.packed_rows(v), L.packed_rows(out)
    B, Hq, Sq, D = q.shape
    need = _workspace_bytes(B, Hq, k.shape[1], Sq, k.shape[2], D, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with L.on_device(dev):
        L.check(L.lib().lcbsa_dense_attn_fwd(qd, kd, vd, shape.packed(), od, None if lse is None else lse.data_ptr(),
                                             None if rest is None else rest.data_ptr(), None if ws is None else ws.data_ptr(), need,
                                             L.current_stream(dev)))
    return out, lse, rest


class _DenseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, shape, return_lse):
        out, lse, rest = _forward(q, k, v, shape, True, True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.rest, ctx.shape = rest, shape
        if not return_lse:
            return out
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, *_):
        q, k, v, out, lse = ctx.saved_tensors
        dev = q.device
        dq, dk, dv = (torch.empty_like(t, memory_format=_DENSE) for t in (q, k, v))
        (q, qd), (k, kd), (v, vd), (out, od), (dout, gd) = map(L.packed_rows, (q, k, v, out, dout))
        (_, dqd), (_, dkd), (_, dvd) = map(L.packed_rows, (dq, dk, dv))
        B, Hq, Sq, D = q.shape
        need = _workspace_bytes(B, Hq, k.shape[1], Sq, k.shape[2], D, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        with L.on_device(dev):
            L.check(L.lib().lcbsa_dense_attn_bwd(qd, kd, vd, od, gd, ctx.shape.packed(), lse.data_ptr(), ctx.rest.data_ptr(), dqd, dkd, dvd,
                                                 ws.data_ptr(), need, L.current_stream(dev)))
        return dq, dk, dv, None, None


@torch.compiler.disable
def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, softcap: float = 0.0,
                    slopes: Optional[torch.Tensor] = None, cu_q: Optional[torch.Tensor] = None, cu_k: Optional[torch.Tensor] = None,
                    k_lens: Optional[torch.Tensor] = None, prefix_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(x) v over the keys that a query sees, x_ij = cap tanh(scale q_i k_j / cap) - slope |pos_i - j|.

    ``q [B, Hq, Sq, D]``, ``k``, ``v`` ``[B, Hk, Sk, D]``, bf16 or fp16, D 64 or 128, Hq a multiple of Hk (query head h reads key head
    ``h // (Hq // Hk)``), any strides with D contiguous.  ``scale`` defaults to ``D ** -0.5``; ``softcap`` 0 caps nothing;
    ``slopes [Hq]`` (constants) weigh the distance between the query's place among the keys and the key.

    Which keys a query sees: all of its batch entry's; with ``k_lens [B]`` the first that many (a padded cache); with ``cu_q``
    (``[docs + 1]`` for all entries or ``[B, docs + 1]``, the first token of every document and the end of the last) and ``cu_k`` (default
    ``cu_q``) those of its own document, none if it belongs to none.  The last query of a document (of an entry) stands at its last key;
    ``causal`` hides the keys behind a query's place, except the first ``prefix_lens`` (``[docs]`` or ``[B, docs]``, docs 1 without
    ``cu_q``) of the document.  These numbers stay on the GPU: nothing is read back, and a captured call replays with what they then
    hold.  A query that sees nothing gets 0 (``lse`` -inf).  What is hidden may hold anything, infinities and NaN included.

    Returns ``out [B, Hq, Sq, D]``, with ``return_lse`` also the fp32 ``lse [B, Hq, Sq]`` (no gradient runs through it)."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("dense_attention needs CUDA tensors; there is no CPU path")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("expected q [B, Hq, Sq, D] and k, v [B, Hk, Sk, D]")
    if k.device != q.device or v.device != q.device:
        raise ValueError(f"q, k, v are on {q.device}, {k.device}, {v.device}")
    shape = _shape_of(q, k, causal, softcap, slopes, cu_q, cu_k, k_lens, prefix_lens, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _DenseAttention.apply(q, k, v, shape, return_lse)
    out, lse, _ = _forward(q, k, v, shape, return_lse)
    return (out, lse) if return_lse else out
