"""Linear attention with a decay for each head: chunked over a prompt, recurrent for single tokens.

With ``lambda_h = exp(log_decay[h])``::

    S_t = lambda S_{t-1} + k_t v_t^T            y_t = scale * q_t^T S_t

so ``y_t = scale * sum_{n<=t} lambda^(t-n) (q_t . k_n) v_n``.  The reference has the form without a decay, a state or a
backward (``CausalLinear``, lra/models/triton/causal_linear.py:23-145; ``causal_linear`` here).  ``decay_linear`` is the
training form, ``decay_linear_prefill`` and ``decay_linear_decode`` the serving pair over a state fp32 [B, H, Dk, Dv].

q, k: [B,H,N,Dk], v: [B,H,N,Dv] in one of fp32, fp16, bf16, any strides (the 'b n (h d) -> b h n d' views of the modules are
taken as they are); Dk, Dv up to 256.  ``log_decay``: [H], a constant of the model (no gradient), usually at most 0: 0 is no
decay, -inf leaves a token itself alone.  ``lengths``: int32 (or int64) [B]; tokens at or behind ``lengths[b]`` -- padding,
which may hold anything -- leave the state alone and have outputs and gradients of zero.  A value that is not finite among the
live tokens spoils the outputs of the 128-token chunk it stands in, also those before it.  Products, weighted values and states of
fp16 operands carry powers of two of their own, so that small and large ones keep their bits; results are fp16's.  Weighted
products of one token that are 2^37 times smaller than its largest do not (under strong growth, where what is large meets zeros in v).
"""
from __future__ import annotations

import torch

from ._cabi import native
from .mixer import _autocast, _need_cuda, ops

__all__ = ["decay_linear", "decay_linear_prefill", "decay_linear_decode", "decay_linear_state_init"]


def decay_linear_state_init(B: int, H: int, Dk: int, Dv: int, device) -> torch.Tensor:
    """The state of an empty prefix."""
    return torch.zeros(B, H, Dk, Dv, dtype=torch.float32, device=device)


def decay_linear(q, k, v, log_decay, scale: float = 1.0, lengths=None):
    """y [B,H,N,Dv] of a whole sequence from an empty state; differentiable in q, k and v.

    A second derivative and forward mode raise.  Nothing of the forward but its operands is kept for the backward.  Works under torch.autocast (q, k, v are cast to the
    autocast dtype) and inside torch.compile (registered operators ``flare_b200::decay_fwd`` / ``decay_bwd``)."""
    q, k, v = _autocast(q, k, v)
    if torch.compiler.is_compiling():
        _need_cuda(q, k, v)
        return ops.decay_fwd(q, k, v, log_decay, float(scale), lengths)
    return native.decay(q, k, v, log_decay, float(scale), lengths)


def decay_linear_prefill(q, k, v, log_decay, scale: float = 1.0, state=None, lengths=None):
    """(y [B,H,N,Dv], state after the last live token) from ``state`` (None: empty), which is left as it is.  Forward only.

    The state is as exact as sums in 32 bits for values of like size along a sequence.  Padding belongs into ``lengths``: behind
    tokens that were silenced by zeros in k instead, a 16-bit call keeps less of what came before them."""
    q, k, v = _autocast(q, k, v)
    return native.decay_prefill(q, k, v, log_decay, float(scale), state, lengths)


def decay_linear_decode(q, k, v, log_decay, state, scale: float = 1.0, lengths=None):
    """The tokens of q, k, v (N is usually 1) one after the other; ``state`` is updated in place.  Forward only.

    A sequence of length 0 sits the call out: its state stays, its outputs are zero."""
    q, k, v = _autocast(q, k, v)
    return native.decay_decode(q, k, v, log_decay, state, float(scale), lengths)


@torch.library.register_fake("flare_b200::decay_fwd")
def _(q, k, v, log_decay, scale, lengths):
    return _like_rows(v)


@torch.library.register_fake("flare_b200::decay_bwd")
def _(q, k, v, dy, log_decay, scale, lengths):
    return _like_rows(q), _like_rows(k), _like_rows(v)


def _like_rows(t):
    """What the kernels return beside t: t's strides when it is dense with a unit last stride and addressable, else row-major."""
    rows = t.contiguous() if t.stride(-1) != 1 and t.shape[-1] != 1 else t
    if rows.element_size() == 2 and rows.shape[-1] % 8 == 0 and \
            any((s * 2) % 16 or (s == 0 and n != 1) for s, n in zip(rows.stride()[:-1], rows.shape[:-1])):
        rows = rows.contiguous()
    out = torch.empty_like(rows)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)
