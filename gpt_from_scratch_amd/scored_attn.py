"""Attention whose scores are capped, biased by distance or masked by documents or
a prefix, with key heads shared by query heads; and its form for single tokens.

``scored_attn(q, k, v, causal=True, ...)`` takes q ``[B, H, Sq, D]`` and k, v
``[B, Hk, Sk, D]`` (any strides; H a multiple of Hk, Sq <= Sk: the queries are the
last Sq of the Sk positions) and returns a contiguous ``[B, H, Sq, D]``:

* ``softcap=c``: scores ``z = softmax_scale * q.k`` become ``c * tanh(z / c)``;
* ``slopes`` (fp32 ``[H]``, not trained): then ``z - slopes[h] * |i - j|``;
* ``document_ids`` (int32 ``[B, Sk]``): a query sees only keys of its own
  document; negative ids are padding, which sees nothing, is seen by nothing and
  may hold anything.  Ids need not be sorted, tiles are skipped where they are;
* ``causal``: a query sees keys up to its own position, and with ``prefix_lens``
  (int32 ``[B]``) also the first ``prefix_lens[b]`` keys.

A query that sees no key gets zeros (lse -inf) and passes no gradient.  Masked keys
outside the padding must be finite, as for ``apply_flash_attn``.  fp32, fp16 and
bf16; D a multiple of 8 up to 128.  The backward gives dq, dk and dv (dk and dv
summed over the query heads of each key head) without atomics.

``decode_attn(q, k, v, lengths=None, ...)`` is the newest token of each sequence
over its cache: q ``[B, H, D]``, k and v ``[B, Hk, S, D]``, the first ``lengths[b]``
(int32 ``[B]``; all S without) of them filled and the token the last of these.  It
has no backward.

The reference's attention (core/myFlashAttn.py:198-441) has none of the
modifications, and as many key heads as query heads.
"""
from __future__ import annotations

import math

import torch

from . import _lib

MAX_KEYS = 1 << 24


def _check_heads(q, k, v, q_dims, what):
    if q.dim() != q_dims or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"{what}; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, H, D = q.shape[0], q.shape[1], q.shape[-1]
    if k.shape[0] != B or k.shape[3] != D or 0 in q.shape or 0 in k.shape or H % k.shape[1]:
        raise ValueError(f"{what}, H a multiple of Hk, no size 0; got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q, k, v must share a dtype; got {q.dtype}, {k.dtype}, {v.dtype}")
    _lib.dtype_code(q)
    if D % 8 or D > 128:
        raise ValueError(f"head dim {D}: a multiple of 8 up to 128")
    if k.shape[2] > MAX_KEYS:
        raise ValueError(f"{k.shape[2]} keys: at most {MAX_KEYS}")


def _check_scores(q, softcap, slopes, scale):
    if softcap is not None and not 1e-6 <= softcap <= 1e4:
        raise ValueError(f"softcap must be between 1e-6 and 1e4 (or None), got {softcap}")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"softmax_scale must be positive and finite, got {scale}")
    if slopes is not None:
        if slopes.dtype != torch.float32 or tuple(slopes.shape) != (q.shape[1],):
            raise ValueError(f"slopes must be float32 [{q.shape[1]}]; got {slopes.dtype} "
                             f"{tuple(slopes.shape)}")


def _check_slopes_grad(slopes):
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("slopes take no gradient: detach them")


def _check_ints(name, t, shape):
    if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != shape):
        raise ValueError(f"{name} must be int32 {list(shape)}; got {t.dtype} {tuple(t.shape)}")


def _check(q, k, v, causal, softcap, slopes, document_ids, prefix_lens, scale):
    _check_heads(q, k, v, 4, "q must be [B, H, Sq, D] and k, v [B, Hk, Sk, D]")
    B, Sq, Sk = q.shape[0], q.shape[2], k.shape[2]
    if Sq > Sk:
        raise ValueError(f"more queries ({Sq}) than keys ({Sk})")
    _check_scores(q, softcap, slopes, scale)
    _check_ints("document_ids", document_ids, (B, Sk))
    _check_ints("prefix_lens", prefix_lens, (B,))
    if prefix_lens is not None and not causal:
        raise ValueError("prefix_lens: with causal only")
    _lib._require_gpu(q, k, v, *(t for t in (slopes, document_ids, prefix_lens) if t is not None))


def _dense(t):
    return None if t is None else t.contiguous()


def _scale(q, scale):
    return 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)


def _forward(q, k, v, causal, softcap, slopes, document_ids, prefix_lens, scale, grad=False):
    _check(q, k, v, causal, softcap, slopes, document_ids, prefix_lens, scale)
    q, k, v = (_lib.rows_ready(t) for t in (q, k, v))
    mods = (bool(causal), softcap, _dense(slopes), _dense(document_ids), _dense(prefix_lens))
    with torch.cuda.device(q.device):
        return (q, k, v), mods, _lib.sattn_fwd(q, k, v, mods, scale, grad)


class ScoredAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, softcap, slopes, document_ids, prefix_lens, scale):
        qkv, mods, (o, o_lo, lse, tiles) = _forward(q, k, v, causal, softcap, slopes, document_ids,
                                                    prefix_lens, scale, any(ctx.needs_input_grad))
        ctx.save_for_backward(*qkv, o, o_lo, lse, tiles, *mods[2:])
        ctx.meta = mods[0], mods[1], scale
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, o_lo, lse, tiles, slopes, docs, prefix = ctx.saved_tensors
        causal, softcap, scale = ctx.meta
        do = _lib.rows_ready(do.to(q.dtype))
        # what was saved may come back through a saved-tensor hook as something else
        _check(q, k, v, causal, softcap, slopes, docs, prefix, scale)
        if do.shape != q.shape or o.shape != q.shape or o.dtype != q.dtype \
                or lse.shape != q.shape[:3] or lse.dtype != torch.float32 \
                or not all(t.is_contiguous() for t in (o, lse)) \
                or (o_lo is not None and (o_lo.shape != o.shape or o_lo.dtype != o.dtype
                                          or not o_lo.is_contiguous())):
            raise ValueError("the gradient and the saved tensors do not fit each other")
        if docs is not None and (tiles.dtype != torch.int32 or not tiles.is_contiguous()
                                 or tiles.numel() != _lib.sattn_tiles(q, k)):
            raise ValueError("the saved document tiles do not fit")
        q, k, v = (_lib.rows_ready(t) for t in (q, k, v))
        slopes, docs, prefix = _dense(slopes), _dense(docs), _dense(prefix)
        with torch.cuda.device(q.device):
            grads = _lib.sattn_bwd(q, k, v, o, o_lo, do, lse, tiles,
                                   (causal, softcap, slopes, docs, prefix), scale)
        return (*grads, None, None, None, None, None, None)


def scored_attn(q, k, v, causal: bool = True, softcap=None, slopes=None, document_ids=None,
                prefix_lens=None, softmax_scale=None):
    """Attention with modified scores (see the module's text), differentiable in q, k, v."""
    o = _lib.ops().scored_attn(q, k, v, causal, softcap, slopes, document_ids, prefix_lens,
                               softmax_scale)
    if o is not None:
        return o
    _check_slopes_grad(slopes)
    return ScoredAttn.apply(q, k, v, causal, softcap, slopes, document_ids, prefix_lens,
                            _scale(q, softmax_scale))


def scored_attn_forward(q, k, v, causal: bool = True, softcap=None, slopes=None, document_ids=None,
                        prefix_lens=None, softmax_scale=None):
    """Forward only, without autograd: ``(O, lse)``, lse the fp32 ``[B, H, Sq]``
    log-sum-exp of the visible scores."""
    out = _lib.ops().scored_attn_forward(q, k, v, causal, softcap, slopes, document_ids,
                                         prefix_lens, softmax_scale)
    if out is not None:
        return out
    with torch.no_grad():
        o, _, lse, _ = _forward(q, k, v, causal, softcap, slopes, document_ids, prefix_lens,
                                _scale(q, softmax_scale))[2]
        return o, lse


def decode_attn(q, k, v, lengths=None, softcap=None, slopes=None, softmax_scale=None):
    """Attention of one new token of each sequence over its cache: ``[B, H, D]``."""
    o = _lib.ops().decode_attn(q, k, v, lengths, softcap, slopes, softmax_scale)
    if o is not None:
        return o
    scale = _scale(q, softmax_scale)
    _check_heads(q, k, v, 3, "q must be [B, H, D] and k, v [B, Hk, S, D]")
    _check_scores(q, softcap, slopes, scale)
    _check_slopes_grad(slopes)
    _check_ints("lengths", lengths, (q.shape[0],))
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        raise RuntimeError("decode_attn has no backward: call it under torch.no_grad(), or use "
                           "scored_attn")
    _lib._require_gpu(q, k, v, *(t for t in (lengths, slopes) if t is not None))
    with torch.cuda.device(q.device):
        return _lib.decode_attn(*(_lib.rows_ready(t) for t in (q, k, v)), _dense(lengths), softcap,
                                _dense(slopes), scale)
