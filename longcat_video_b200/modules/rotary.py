"""Rotary positions along one axis: interleaved and half layouts, part of the head, frequencies scaled for long contexts.

The 1-D counterpart of the rotary embedding over a latent grid (``rope_3d.py``, longcat_video/modules/rope_3d.py:60-120), for q
and k of a text model in front of ``dense_attention``.  The angles are right to 2^-24 of half a turn up to positions of 2^40 (64-bit
fixed-point turns inside the kernel, see ``csrc/rotary.cu``).  All arithmetic on q and k is in liblcbsa.so (``lcbsa_rotary``); there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
import math
from fractions import Fraction
from typing import Mapping, Optional, Tuple

import torch

from .. import _lib as L


_PI = Fraction("3.14159265358979323846264338327950288419716939937510")


class RotaryFrequencies:
    """``pairs`` frequencies in turns per position, as 64-bit fixed point, and the factor on the result (``rotary_frequencies``)."""

    def __init__(self, radians, factor: float = 1.0):
        self.radians = tuple(float(f) for f in radians)
        self.factor = float(factor)
        self.pairs = len(self.radians)
        if not all(math.isfinite(f) for f in self.radians) or not math.isfinite(self.factor):
            raise ValueError("frequencies and factor must be finite")
        self.turns = (ctypes.c_uint64 * self.pairs)(*(round(Fraction(f) / (2 * _PI) * 2 ** 64) % 2 ** 64 for f in self.radians))
        self.address = ctypes.addressof(self.turns)


_KINDS = {"linear": {"factor"}, "base": {"factor"}, "by_parts": {"factor", "original_length", "fast", "slow", "attention_factor"},
          "by_wavelength": {"factor", "original_length", "low", "high"}}


@functools.lru_cache(maxsize=64)
def _frequencies(rotary_dim: int, base: float, scaling) -> RotaryFrequencies:
    s = dict(scaling)
    kind, factor = s.get("kind"), float(s.get("factor", 1.0))
    if kind is not None:
        if kind not in _KINDS or set(s) - _KINDS[kind] - {"kind"}:
            raise ValueError(f"scaling {s}: one of {sorted(_KINDS)} with its own parameters")
        if not (math.isfinite(factor) and factor >= 1.0):
            raise ValueError(f"scaling factor {factor}: at least 1")
        if "original_length" in _KINDS[kind] and not s.get("original_length", 0) > 0:
            raise ValueError(f"scaling {s}: needs the original_length, a positive number")
    if kind == "base":
        if rotary_dim == 2:
            raise ValueError("scaling by the base needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pairs = rotary_dim // 2
    f = [base ** (-2 * i / rotary_dim) for i in range(pairs)]
    result = 1.0
    if kind == "linear":
        f = [x / factor for x in f]
    elif kind == "by_parts":
        length, fast, slow = float(s["original_length"]), float(s.get("fast", 32.0)), float(s.get("slow", 1.0))
        at = lambda turns: rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(pairs)]
        f = [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)]
        given = s.get("attention_factor")
        result = 0.1 * math.log(factor) + 1.0 if given is None else float(given)
    elif kind == "by_wavelength":
        length, low, high = float(s["original_length"]), float(s.get("low", 1.0)), float(s.get("high", 4.0))
        if not high > low:
            raise ValueError(f"scaling by wavelength needs high {high} above low {low}")
        keep = [min(max((length * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        f = [x / factor * (1 - s_) + x * s_ for x, s_ in zip(f, keep)]
    return RotaryFrequencies(f, result)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[Mapping] = None) -> RotaryFrequencies:
    """Frequencies ``base ** (-2 i / rotary_dim)`` radians per position of the ``rotary_dim / 2`` pairs (``rotary_dim`` a multiple of
    16 up to 256), scaled for contexts ``factor`` times as long as a model was trained on:

    ``{"kind": "linear", "factor": s}``  all frequencies divided by s
    ``{"kind": "base", "factor": s}``  base times ``s ** (r / (r - 2))``: the lowest frequency divided by s, the highest as it is
    ``{"kind": "by_parts", "factor": s, "original_length": n}``  pairs that turn more than ``fast`` (32) times in n positions stay, those
    below ``slow`` (1) are divided by s, a ramp over the pair's number between them; q and k are multiplied by ``attention_factor``
    (default ``0.1 ln s + 1``)
    ``{"kind": "by_wavelength", "factor": s, "original_length": n}``  pairs with more than ``high`` (4) turns in n positions stay, those below
    ``low`` (1) are divided by s, a ramp over the turns between them

    A pure function of its arguments; the last 64 results are kept."""
    if rotary_dim < 16 or rotary_dim > 256 or rotary_dim % 16:
        raise ValueError(f"rotary_dim {rotary_dim}: a multiple of 16 in 16 .. 256")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"base {base}: a number above 1")
    return _frequencies(int(rotary_dim), float(base), tuple(sorted((scaling or {}).items())))


def _embed(xs, freqs, positions, offset, interleaved):
    x0 = xs[0]
    for x in xs:
        if not x.is_cuda:
            raise RuntimeError("the rotary embedding needs CUDA tensors; there is no CPU path")
        if x.dim() != 4:
            raise ValueError("expected [B, H, S, D] tensors")
        if x.device != x0.device:
            raise ValueError(f"tensors on {x0.device} and {x.device}")
        L.dtype_code(x.dtype)
        if 2 * freqs.pairs > x.shape[3]:
            raise ValueError(f"{2 * freqs.pairs} turning dimensions of a head of {x.shape[3]}")
    B, _, S, _ = x0.shape
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, not {positions.dtype}")
        if positions.device != x0.device:
            raise ValueError(f"positions on {positions.device}, the tensors on {x0.device}")
        if tuple(positions.shape) not in ((S,), (1, S), (B, S)):
            raise ValueError(f"positions of shape {tuple(positions.shape)} for {B} entries of {S} tokens")
        if offset:
            raise ValueError("positions and offset exclude each other")
    return L.binding().rotary(xs, freqs.address, freqs.pairs, freqs.factor, positions, int(offset), interleaved)


@torch.compiler.disable
def embed_rotary(x: torch.Tensor, freqs: RotaryFrequencies, positions: Optional[torch.Tensor] = None, *, offset: int = 0,
                 interleaved: bool = False) -> torch.Tensor:
    """The rows of ``x [B, H, S, D]`` (bf16 or fp16, any strides with D contiguous, D a multiple of 8) with the first ``2 * freqs.pairs``
    dimensions turned by their positions: pairs ``(2p, 2p + 1)`` if ``interleaved``, else ``(p, p + pairs)``; the rest of the head is
    copied.  ``positions``: int32 or int64 ``[S]`` or ``[B, S]`` on the GPU, of any sign, the angles of those beyond 2^40 in size off by
    ``|position| * 2^-65`` turns; without them token s stands at ``offset + s``."""
    return _embed((x,), freqs, positions, offset, interleaved)[0]


@torch.compiler.disable
def embed_rotary_qk(q: torch.Tensor, k: torch.Tensor, freqs: RotaryFrequencies, positions: Optional[torch.Tensor] = None, *, offset: int = 0,
                    interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``embed_rotary`` of a layer's q and k (any numbers of heads) in one launch."""
    return _embed((q, k), freqs, positions, offset, interleaved)
