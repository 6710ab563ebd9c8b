"""Rotary embedding in the forms ``apply_rope_qk`` does not have, alone and behind
the norm of each query and key head.

``apply_rotary_qk(q, k, cos, sin, positions=None, interleaved=True)`` turns the
first ``2 * cos.shape[1]`` elements of each head of q ``[S, B, H, D]`` and k
``[S, B, Hk, D]`` (any strides) and copies the rest:

* pairs ``(2i, 2i + 1)`` (``interleaved``, as ``apply_rope_qk``) or ``(i, i + n)``
  with ``n = cos.shape[1]``;
* the angles of token ``(s, b)`` are row ``positions[s]`` or ``positions[s, b]`` of
  the tables (int32 or int64 positions: packed documents, decoding), row ``s``
  without positions.  A position that the tables do not have gives NaN.

``qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, ...)`` first normalises every
head, ``n = x * rsqrt(mean(x^2) + eps) * weight`` over its D elements, then turns n:
one pass over q and k forward, one backward (and the sum of the weights'
gradients).  Both compute in fp32 and round once.  Tables for long contexts come
from ``RotaryEmbedding(..., scaling=RotaryScaling(...))``; ``RotaryEmbedding(2 * n)``
gives those of a part of the head.

The reference has the interleaved rotation of whole heads at positions
``0 .. S - 1`` (core/rope_triton.py:10-148).
"""
from __future__ import annotations

import torch

from . import _lib

MAX_NORM_DIM = 512


def _check(q, k, cos, sin, positions):
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q must be [S, B, H, D] and k [S, B, Hk, D]; got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if q.dtype != k.dtype:
        raise TypeError(f"q and k must share a dtype; got {q.dtype}, {k.dtype}")
    _lib.dtype_code(q)
    S, B, _, D = q.shape
    if 0 in q.shape or 0 in k.shape:
        raise ValueError(f"q and k must not be empty; got {tuple(q.shape)}, {tuple(k.shape)}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype:
        raise ValueError(f"cos and sin must be [positions, angles] of one shape and dtype; got "
                         f"{tuple(cos.shape)} {cos.dtype}, {tuple(sin.shape)} {sin.dtype}")
    _lib.dtype_code(cos)
    if not 1 <= cos.shape[1] <= D // 2:
        raise ValueError(f"{cos.shape[1]} angles do not fit a head of {D} elements")
    if positions is None:
        if cos.shape[0] < S:
            raise ValueError(f"tables of {cos.shape[0]} rows for {S} positions")
        return
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if tuple(positions.shape) not in ((S,), (S, B)):
        raise ValueError(f"positions must be [{S}] or [{S}, {B}]; got {tuple(positions.shape)}")
    if cos.shape[0] == 0:
        raise ValueError("tables without rows")


def _check_norm(q, q_weight, k_weight, eps):
    D = q.shape[3]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if tuple(w.shape) != (D,):
            raise ValueError(f"{name} must be [{D}]; got {tuple(w.shape)}")
        _lib.dtype_code(w)
    if q_weight.dtype != k_weight.dtype:
        raise TypeError(f"the weights must share a dtype; got {q_weight.dtype}, {k_weight.dtype}")
    if D > MAX_NORM_DIM:
        raise ValueError(f"head dim {D}: at most {MAX_NORM_DIM} with the norm")


def _like(t):
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


class RotaryQK(torch.autograd.Function):
    """q and k turned; the backward turns their gradients back."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved: bool):
        _check(q, k, cos, sin, positions)
        _lib._require_gpu(q, k, cos, sin, *([] if positions is None else [positions]))
        q_out, k_out = _like(q), _like(k)
        with torch.cuda.device(q.device):
            _lib.rotary_qk(q, k, cos, sin, positions, interleaved, q_out, k_out, inverse=False)
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved = interleaved
        return q_out, k_out

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        _check(gq, gk, cos, sin, positions)
        dq, dk = _like(gq), _like(gk)
        with torch.cuda.device(gq.device):
            _lib.rotary_qk(gq, gk, cos, sin, positions, ctx.interleaved, dq, dk, inverse=True)
        return dq, dk, None, None, None, None


class QKNormRotary(torch.autograd.Function):
    """q and k normalised head by head and turned."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, interleaved: bool, eps: float):
        _check(q, k, cos, sin, positions)
        _check_norm(q, q_weight, k_weight, eps)
        _lib._require_gpu(q, k, q_weight, k_weight, cos, sin,
                          *([] if positions is None else [positions]))
        wq, wk = q_weight.contiguous(), k_weight.contiguous()
        q_out, k_out = _like(q), _like(k)
        with torch.cuda.device(q.device):
            _lib.qk_norm_rotary(q, k, wq, wk, cos, sin, positions, interleaved, eps, q_out, k_out)
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        ctx.meta = interleaved, eps
        return q_out, k_out

    @staticmethod
    def backward(ctx, gq, gk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        interleaved, eps = ctx.meta
        _check(gq, gk, cos, sin, positions)
        if q.shape != gq.shape or k.shape != gk.shape or q.dtype != gq.dtype:
            raise ValueError("the gradients do not match q and k")
        dq, dk, dwq, dwk = (_like(t) for t in (q, k, wq, wk))
        with torch.cuda.device(q.device):
            _lib.qk_norm_rotary_bwd(q, k, wq, wk, cos, sin, positions, interleaved, eps, gq, gk,
                                    dq, dk, dwq, dwk)
        return dq, dk, dwq, dwk, None, None, None, None, None


def apply_rotary_qk(q, k, cos, sin, positions=None, interleaved: bool = True):
    """``(q', k')``: q ``[S, B, H, D]`` and k ``[S, B, Hk, D]`` turned by the tables'
    angles (see the module's text)."""
    out = _lib.ops().rotary_qk(q, k, cos, sin, positions, interleaved)
    if out is None:
        return RotaryQK.apply(q, k, cos, sin, positions, bool(interleaved))
    return out


def qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, eps: float = 1e-6, positions=None,
                   interleaved: bool = True):
    """``apply_rotary_qk`` of the heads' RMSNorm with weights ``[D]``, in one pass."""
    out = _lib.ops().qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps)
    if out is None:
        return QKNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, bool(interleaved),
                                  float(eps))
    return out
