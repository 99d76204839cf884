"""Sequence operators beside the signature layers: decayed linear attention over the time axis and the norm around a
block.

A signature folds a time-ordered sequence into iterated outer products; the layers here mix a sequence of such features
(for example the ``(B, W, D)`` windows of :class:`Signature`) over time.  The state of :func:`linear_attention` is the
degree-2 tensor of its keys and values with a fading memory -- without decay, with ``k_t = x_{t-1} - x_0 + dx_t / 2``
and ``v_t = dx_t``, it is the second degree of the signature of ``x`` -- and :func:`linear_attention_step` updates it by
one time step, as :func:`chen_product` extends a signature.  :func:`gated_residual_norm` brings rows to one scale around a
block; its weight lets features of different size (signature words shrink with 1/degree!) count as the model learns.  The reference package has no counterpart.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import ops

_ACTIVATIONS = {"silu": 0, "sigmoid": 1}


def _scale(q: Tensor, scale: Optional[float]) -> float:
    if scale is None:
        return q.shape[-1] ** -0.5 if q.dim() > 0 and q.shape[-1] > 0 else 1.0
    if isinstance(scale, Tensor) or not math.isfinite(scale):
        raise ValueError("scale must be a finite number")
    return float(scale)


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, *, initial_state: Optional[Tensor] = None,
                     lengths: Optional[Tensor] = None, scale: Optional[float] = None, return_state: bool = False):
    """Causal linear attention with a decay for each head, over whole sequences.

    Per sequence and head, from ``S = initial_state`` (zeros by default)::

        S_t = exp(log_decay_t) * S_{t-1} + k_t v_t^T,        out_t = scale * S_t^T q_t

    ``q`` (B, L, H, Dk), ``k`` (B, L, Hkv, Dk), ``v`` (B, L, Hkv, Dv): float32, float64, bfloat16 or float16, any
    strides; H is a multiple of Hkv and consecutive heads of ``q`` share a head of ``k`` and ``v``.  Head sizes are at
    most 256.  ``log_decay``: float32 (float64 for float64 operands), (H) -- a constant per head -- or (B, L, H), for
    example ``-rate * dt`` for irregularly spaced observations.  It is meant to be at most 0 (growth beyond 2^127 within 32
    steps may overflow where the results do not); ``-inf`` forgets all that was before the step.  ``initial_state`` (B, H, Dk, Dv): the type of ``log_decay``.  ``lengths`` (B), int32 or int64
    on the GPU: later rows of a sequence are not read, their output is 0, and the state stops there (values outside
    [0, L] are clamped).  Rows up to the lengths are meant to be finite: an infinity or NaN there may reach every step of its
    sequence and head, steps up to 127 before it too.  ``scale`` defaults to ``Dk ** -0.5``.

    Returns the output (B, L, H, Dv) in the type of ``q``; with ``return_state`` also the state after the last step
    (B, H, Dk, Dv).  Differentiable once wrt all floating operands (second derivatives and forward mode are
    refused); gradients are the same bits on every run.  Under CUDA graph capture, capture forward and backward together, with no graph of an
    eager call on the same leaves alive.
    """
    out, state = ops.linear_attention(q, k, v, log_decay, initial_state, lengths, _scale(q, scale), bool(return_state))
    return (out, state) if return_state else out


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *,
                          scale: Optional[float] = None) -> Tensor:
    """One time step of :func:`linear_attention` for every sequence, on a kept state.

    ``q`` (B, H, Dk), ``k`` (B, Hkv, Dk), ``v`` (B, Hkv, Dv), ``log_decay`` (H) or (B, H); ``state`` (B, H, Dk, Dv),
    contiguous, in the type of ``log_decay``, is updated in place (a graph that has saved it then refuses its backward
    pass).  Returns the output (B, H, Dv).  For serving: not
    differentiable.
    """
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError("linear_attention_step is not differentiable; call it under torch.no_grad(), or use "
                           "linear_attention with L = 1")
    return ops.linear_attention_step(q, k, v, log_decay, state, _scale(q, scale))


def gated_residual_norm(x: Tensor, weight: Optional[Tensor] = None, *, gate: Optional[Tensor] = None,
                        activation: str = "silu", residual: Optional[Tensor] = None,
                        residual_scale: Optional[Tensor] = None, next_weight: Optional[Tensor] = None,
                        eps: float = 1e-6):
    """The norm after a block with the block's gate, the scaled residual sum and the norm before the next block.

    Over the last dimension of ``x`` (..., D), with ``rms(x) = x / sqrt(mean(x^2) + eps)``::

        h = residual + residual_scale * (rms(x) * weight * act(gate)),       n = rms(h) * next_weight

    Operands left out drop their factor or term; ``act(g)`` is ``g * sigmoid(g)`` ("silu") or ``sigmoid(g)``
    ("sigmoid").  ``x``, ``gate`` and ``residual`` share shape and type (float32, float64, bfloat16 or float16);
    ``weight``, ``residual_scale`` and ``next_weight`` (D) are float32 (float64 next to float64), or in the type of
    ``x``.  ``n`` is the norm of h before h is rounded.

    Returns ``h``, or ``(h, n)`` when ``next_weight`` is given, in the type of ``x``.  Differentiable once wrt all
    operands (second derivatives and forward mode are refused); gradients are the same bits on every run.
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}")
    if not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    weight, residual_scale, next_weight = (
        t.to(torch.float32) if t is not None and t.dtype == x.dtype and x.dtype in (torch.bfloat16, torch.float16) else t
        for t in (weight, residual_scale, next_weight))
    h, n = ops.gated_residual_norm(x, weight, gate, residual, residual_scale, next_weight, _ACTIVATIONS[activation],
                                   float(eps))
    return (h, n) if next_weight is not None else h
