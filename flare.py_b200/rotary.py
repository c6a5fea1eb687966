"""Rotary positions of queries and keys.

``rotary(x, freqs)`` turns the pair (x0, x1) of a head's features by the angle ``position * freqs[i]``::

    (x0, x1)  ->  scale * (x0 cos - x1 sin, x0 sin + x1 cos)

for the first R = 2 * len(freqs) features: pairs (i, i + R/2), or (2 i, 2 i + 1) when ``interleaved``; the others pass
through.  Angles are formed in 64 bits, so far positions lose nothing.  The reference rotates k in its lra blocks
(lra/models/embeddings.py, lra/models/backends.py:599-600); ``Rotary`` is what ``LraFLARE(rope=...)`` takes.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import nn

from ._cabi import native
from .mixer import _need_cuda, ops

__all__ = ["rotary", "rotary_pair", "rotary_frequencies", "Rotary"]


def rotary_frequencies(dim: int, base: float = 10_000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, turns: Tuple[float, float] = (1.0, 32.0)) -> Tuple[torch.Tensor, float]:
    """(freqs fp64 [dim/2] on the CPU, the ``scale`` that goes with them) for `dim` rotated features.

    scaling: None         base^(-2i/dim)
             "linear"     the same over `factor`: positions are squeezed into the trained range
             "ntk"        base * factor^(dim/(dim-2)): the slowest pair is slowed by `factor`, the fastest stays
             "by_parts"   pairs that turn fewer than turns[0] times over `original_length` are slowed by `factor`, those above
                          turns[1] stay, a linear ramp between; scale 1 + 0.1 ln(factor)   (YaRN, arXiv:2309.00071)"""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be an even number of features, got {dim}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    exponent = torch.arange(0, dim, 2, dtype=torch.float64, device="cpu") / dim
    freqs = base ** -exponent
    if scaling is None:
        if factor != 1.0:
            raise ValueError("a factor needs a scaling: 'linear', 'ntk' or 'by_parts'")
        return freqs, 1.0
    if scaling == "linear":
        return freqs / factor, 1.0
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("scaling 'ntk' needs at least four features")
        return (base * factor ** (dim / (dim - 2))) ** -exponent, 1.0
    if scaling == "by_parts":
        if original_length is None or original_length < 1:
            raise ValueError("scaling 'by_parts' needs the original_length")
        slow, fast = turns
        if not slow < fast:
            raise ValueError(f"turns must ascend, got {turns}")
        keep = ((original_length * freqs / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        return freqs * keep + freqs / factor * (1.0 - keep), (1.0 + 0.1 * math.log(factor) if factor > 1.0 else 1.0)
    raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'by_parts', got {scaling!r}")


def rotary(x, freqs, positions=None, offset: int = 0, interleaved: bool = False, scale: float = 1.0):
    """x [B,H,N,D] (fp32, fp16 or bf16, any strides) with its first 2 * len(freqs) features turned; differentiable by
    torch.autograd, any number of times, and in forward mode (torch.func's reverse-mode transforms take no native autograd function
    and raise).  freqs: fp64 on x's device.  Token n stands at ``positions[n]`` (int32 or int64; [N], [1,N] or [B,N]) or, without
    positions, at n; ``offset`` is added to either."""
    if torch.compiler.is_compiling():
        _need_cuda(x)
        return ops.rotary(x, freqs, positions, int(offset), bool(interleaved), float(scale), False)
    return native.rotary(x, freqs, positions, int(offset), bool(interleaved), float(scale))


def rotary_pair(q, k, freqs, positions=None, offset: int = 0, interleaved: bool = False, scale: float = 1.0):
    """``rotary`` of q [B,Hq,N,D] and k [B,Hk,N,D] in one launch, the angles computed once for both."""
    if torch.compiler.is_compiling():
        _need_cuda(q, k)
        return ops.rotary_pair(q, k, freqs, positions, int(offset), bool(interleaved), float(scale), False)
    return native.rotary_pair(q, k, freqs, positions, int(offset), bool(interleaved), float(scale))


class Rotary(nn.Module):
    """Rotary positions as a module: ``Rotary(dim)(x)`` for one tensor, ``.pair(q, k)`` for two.  `dim` features of every head
    are turned; the other arguments are those of ``rotary_frequencies``.  The frequencies stay fp64 whatever the module is
    cast to, and are no part of the state dict."""

    def __init__(self, dim: int, base: float = 10_000.0, interleaved: bool = False, scaling: Optional[str] = None,
                 factor: float = 1.0, original_length: Optional[int] = None, turns: Tuple[float, float] = (1.0, 32.0)):
        super().__init__()
        freqs, self.scale = rotary_frequencies(dim, base, scaling, factor, original_length, turns)
        self.interleaved = bool(interleaved)
        self._freqs64 = freqs                                  # on the CPU, wherever the module is built
        self.register_buffer("freqs", freqs.clone().to(torch.empty(0).device), persistent=False)

    def _apply(self, fn, recurse=True):
        before = self.freqs
        super()._apply(fn, recurse)
        # A cast must not round them, nor to_empty leave them unset; where nothing moves, the buffer stays: captured graphs read it.
        stays = self.freqs.device == before.device and before.device.type != "meta"
        self.freqs = before if stays else self._freqs64.to(self.freqs.device, copy=True)
        return self

    def forward(self, x, positions=None, offset: int = 0):
        return rotary(x, self.freqs, positions, offset, self.interleaved, self.scale)

    def pair(self, q, k, positions=None, offset: int = 0):
        return rotary_pair(q, k, self.freqs, positions, offset, self.interleaved, self.scale)


def _like(t):
    rows = t.contiguous() if t.stride(-1) != 1 and t.shape[-1] != 1 else t
    out = torch.empty_like(rows)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


@torch.library.register_fake("flare_b200::rotary")
def _(x, freqs, positions, offset, interleaved, scale, back):
    return _like(x)


@torch.library.register_fake("flare_b200::rotary_pair")
def _(q, k, freqs, positions, offset, interleaved, scale, back):
    return _like(q), _like(k)
