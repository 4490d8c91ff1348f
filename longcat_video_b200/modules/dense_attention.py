"""Dense attention with capped or distance-biased scores and document, prefix and length masks.

What stands beside the block-sparse attention of the DiT: its cross-attention from the video tokens to packed prompts
(``MultiHeadCrossAttention`` with ``kv_seqlen``, longcat_video/modules/attention.py:184-260, a document mask), its
self-attention with block sparsity off (attention.py:67-104), a text encoder whose scores fall off in a line with the distance, an
autoregressive model that shares the GPU.  Forward, backward, and a form for a few tokens of every sequence behind a long cache.
All arithmetic is in liblcbsa.so (``lcbsa_dense_attn_fwd`` / ``_bwd``), which ``csrc/binding.cpp`` calls; there is no CPU path.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import _lib as L


def _numbers(name: str, t: torch.Tensor, device, shapes) -> torch.Tensor:
    """An int32 tensor of one of the shapes on the call's device, contiguous.  What 32 bits do not hold lies outside of every tensor and becomes the
    nearest number that they hold."""
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, q on {device}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {' or '.join(map(str, shapes))}")
    if t.dtype == torch.int64:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _shape_of(q, k, causal, softcap, slopes, cu_q, cu_k, k_lens, prefix_lens, scale) -> tuple:
    """The scores as the binding takes them: (scale, cap, causal, slopes, cu_q, cu_k, k_lens, prefix), checked."""
    B, Hq, _, D = q.shape
    dev = q.device
    softcap = float(softcap)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not math.isfinite(softcap) or softcap < 0:
        raise ValueError(f"softcap {softcap}: 0 (none) or a positive number")
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale} is not finite")
    if abs(scale) > 2.0 ** 126 or softcap > 2.0 ** 126:
        raise ValueError(f"scale {scale}, softcap {softcap}: up to 2^126")
    if softcap and scale and not 2.0 ** -20 <= abs(scale) / softcap <= 2.0 ** 20:
        raise ValueError(f"softcap {softcap}: further than a factor of 2^20 from scale {scale}")
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
        if torch.autograd.forward_ad._current_level >= 0 and torch.autograd.forward_ad.unpack_dual(slopes).tangent is not None:
            raise ValueError("slopes are constants: they carry no tangent")
        slopes = slopes.detach().to(torch.float32).contiguous()
    return scale, softcap, bool(causal), slopes, cu_q, cu_k, k_lens, prefix_lens


@torch.compiler.disable
def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, softcap: float = 0.0,
                    slopes: Optional[torch.Tensor] = None, cu_q: Optional[torch.Tensor] = None, cu_k: Optional[torch.Tensor] = None,
                    k_lens: Optional[torch.Tensor] = None, prefix_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    return_lse: bool = False, impl: int = L.ATTN_AUTO) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(x) v over the keys that a query sees, x_ij = cap tanh(scale q_i k_j / cap) - slope |pos_i - j|.

    ``q [B, Hq, Sq, D]``, ``k``, ``v`` ``[B, Hk, Sk, D]``, bf16 or fp16, D 64 or 128, Hq a multiple of Hk (query head h reads key head
    ``h // (Hq // Hk)``), any strides with D contiguous.  ``scale`` defaults to ``D ** -0.5``; ``softcap`` 0 caps nothing,
    others lie within a factor of 2^20 of ``scale``, both up to 2^126;
    ``slopes [Hq]`` (constants, of any sign) weigh the distance between the query's place among the keys and the key: a line in the distance, no
    table over it.

    Which keys a query sees: all of its batch entry's; with ``k_lens [B]`` the first that many (a padded cache); with ``cu_q``
    (``[docs + 1]`` for all entries or ``[B, docs + 1]``, the first token of every document and the end of the last) and ``cu_k`` (default
    ``cu_q``) those of its own document, none if it belongs to none.  The last query of a document (of an entry) stands at its last key;
    ``causal`` hides the keys behind a query's place, except the first ``prefix_lens`` (``[docs]`` or ``[B, docs]``, docs 1 without
    ``cu_q``) of the document.  These numbers stay on the GPU: nothing is read back, and a captured call replays with what they then
    hold.  A query that sees nothing gets 0 (``lse`` -inf).  What is hidden may hold anything, infinities and NaN included.  Bounds in 64 bits are
    cut to 32.

    ``impl`` names the forward kernel (``ATTN_TC``: tcgen05, ``ATTN_MMA``: the one for few queries) where the choice by size is not wanted.

    A call that is recorded for a backward keeps its operands, ``out``, ``lse`` and one more tensor of the size of ``out``: what rounding left of it.

    Returns ``out [B, Hq, Sq, D]``, with ``return_lse`` also the fp32 ``lse [B, Hq, Sq]`` (no gradient runs through it)."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("dense_attention needs CUDA tensors; there is no CPU path")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("expected q [B, Hq, Sq, D] and k, v [B, Hk, Sk, D]")
    if k.device != q.device or v.device != q.device:
        raise ValueError(f"q, k, v are on {q.device}, {k.device}, {v.device}")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"q, k, v have the types {q.dtype}, {k.dtype}, {v.dtype}")
    L.dtype_code(q.dtype)
    return L.binding().dense_attention(q, k, v, *_shape_of(q, k, causal, softcap, slopes, cu_q, cu_k, k_lens, prefix_lens, scale), return_lse, impl)
