"""Attention with scored rules: capped scores, a distance bias, document,
prefix and length masks, without a (query, key) matrix for any of them.

For query i and key j of sequence b and head h::

    x    = scale * q_i . k_j
    s    = softcap * tanh(x / softcap)  (x without a cap)
           - distance_slopes[h] * |i + offset_b - j|
    seen = j < key_lengths[b]
           and (not causal or j <= i + offset_b or j < prefix_lengths[b])
           and documents[b, i] == key_documents[b, j] >= 0

and O is the softmax of s over the keys seen, times V.  A query that sees no key
gets a zero output, an LSE of -inf and no gradient.  Keys from ``key_lengths`` on
and tokens of a negative document reach no result, whatever they hold.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import _lib, _ops
from ..config import DebugConfig
from ..utils import check_numerical_stability, check_tensor_nan_inf

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def check_qkv(q, k, v, what: str) -> None:
    """Shapes, dtypes and devices of q (B, Sq, H, D) and k, v (B, Sk, Hkv, D)."""
    if _ops.host().qkv_ok(q, k, v, _ops.MAX_HEAD_DIM):
        return
    _ops.check_dual(what, q, k, v)
    for t in (q, k, v):
        if not isinstance(t, torch.Tensor):
            raise TypeError("q, k, v must be torch.Tensor instances")
        if t.dim() != 4:
            raise ValueError("Input tensors must be 4-dimensional [batch, seq_len, num_heads, head_dim]")
    B, _, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"incompatible shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if k.shape[2] == 0 or H == 0 or H % k.shape[2] != 0:
        raise ValueError(f"num_heads {H} must be a positive multiple of num_heads_kv {k.shape[2]}")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"dtype must be one of {SUPPORTED_DTYPES} and equal for q, k, v")
    if q.device.type != "cuda" or k.device != q.device or v.device != q.device:
        raise ValueError(f"{what} requires q, k, v on the same GPU device (there is no CPU path)")
    if D == 0 or D > _ops.MAX_HEAD_DIM:
        raise NotImplementedError(f"{what} has no kernel for head_dim {D} (1..{_ops.MAX_HEAD_DIM})")


def check_scale(scale: Optional[float], D: int) -> float:
    if scale is None:
        return D ** -0.5
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"scale must be finite and positive, got {scale}")
    return float(scale)


def check_softcap(softcap: Optional[float], scale: float) -> float:
    if softcap is None:
        return 0.0
    c = float(softcap)
    # below 2^-60 or so the cap's constants would leave the range of float32
    if not math.isfinite(c) or c < 0 or (0 < c < 1e-6) or c > 1e30:
        raise ValueError(f"softcap must be 0 (none) or within [1e-6, 1e30], got {softcap}")
    if c and scale > 1e37 * c:
        raise ValueError(f"scale must be at most 1e37 times softcap, got {scale} and {softcap}")
    return c


def check_slopes(slopes, B: int, H: int, device):
    if slopes is None:
        return None
    if not isinstance(slopes, torch.Tensor):
        raise TypeError("distance_slopes must be a torch.Tensor")
    if slopes.dtype != torch.float32 or tuple(slopes.shape) not in ((H,), (B, H)):
        raise ValueError(f"distance_slopes must be float32 of shape {(H,)} or {(B, H)}, got {slopes.dtype} "
                         f"{tuple(slopes.shape)}")
    if slopes.device != device:
        raise ValueError(f"distance_slopes must be on {device}, got {slopes.device}")
    _ops.check_dual("distance_slopes", slopes)
    return slopes


def _check_documents(docs, name: str, B: int, S: int, device):
    if not isinstance(docs, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if docs.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64, got {docs.dtype}")
    if tuple(docs.shape) not in ((S,), (1, S), (B, S)):
        raise ValueError(f"{name} must have shape {(S,)} or {(B, S)}, got {tuple(docs.shape)}")
    if docs.device != device:
        raise ValueError(f"{name} must be on {device}, got {docs.device}")
    return docs.expand(B, S)


class ScoredAttentionFunction(torch.autograd.Function):
    """Forward and backward of :func:`flash_attention_v100_scored` on checked inputs."""

    @staticmethod
    def forward(ctx, q, k, v, slopes, rules, return_lse):
        o, lse, near = _ops.scored_fwd(q, k, v, rules, True, True)
        ctx.save_for_backward(q, k, v, o, lse, near, slopes, rules.prefix, rules.lens, rules.offsets, rules.q_docs,
                              None if rules.k_docs is rules.q_docs else rules.k_docs)
        ctx.one_docs = rules.k_docs is rules.q_docs
        ctx.rules = (rules.causal, rules.scale, rules.softcap, rules.offset0)
        if return_lse:
            ctx.mark_non_differentiable(lse)
            return o, lse
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output, grad_lse=None):
        # the gradient of the LSE output is ignored, as flash_attention_v100 does
        q, k, v, o, lse, near, slopes, prefix, lens, offsets, q_docs, k_docs = ctx.saved_tensors
        causal, scale, softcap, offset0 = ctx.rules
        if DebugConfig.VALIDATE_OUTPUTS:
            check_tensor_nan_inf(grad_output, "grad_output")
        rules = _ops.Rules(causal, scale, softcap, slopes, prefix, lens, offsets, offset0, q_docs,
                           q_docs if ctx.one_docs else k_docs)
        dq, dk, dv, ds = _ops.scored_bwd(q, k, v, o, grad_output, lse, near, rules,
                                         slopes is not None and ctx.needs_input_grad[3])
        if DebugConfig.VALIDATE_OUTPUTS:
            for t, name in ((dq, "grad_q"), (dk, "grad_k"), (dv, "grad_v"), (ds, "grad_distance_slopes")):
                check_tensor_nan_inf(t, name)
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, ds, None, None


def flash_attention_v100_scored(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    causal: bool = False,
    scale: Optional[float] = None,
    *,
    softcap: Optional[float] = None,
    distance_slopes: Optional[torch.Tensor] = None,
    documents: Optional[torch.Tensor] = None,
    key_documents: Optional[torch.Tensor] = None,
    prefix_lengths: Optional[torch.Tensor] = None,
    key_lengths: Optional[torch.Tensor] = None,
    query_offsets: Union[int, torch.Tensor, None] = None,
    return_softmax_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention with scored rules on q (B, Sq, H, D) and k, v (B, Sk, Hkv, D);
    the formula is in the module docstring.

    ``softcap``: bound of the tanh on the scores (0 or None: none).
    ``distance_slopes``: float32 (H,) or (B, H), differentiable.  Queries may stand
    off the keys: outputs and gradients keep their digits at any distance (the LSE
    holds slope times the distance to the nearest key).
    ``documents``: integer ids (B, Sq) or (Sq,) of the queries' documents and,
    unless ``key_documents`` gives theirs, of the keys'; negative (or past int32):
    padding.
    ``prefix_lengths``: (B,), with ``causal``: keys before them are seen by every
    query.  ``key_lengths``: (B,) filled keys.  ``query_offsets``: position of
    query 0 among the keys, an int or (B,); 0 by default (the top-left causal mask
    of :func:`flash_attention_v100`), ``key_lengths - Sq`` for new tokens at the
    end of a cache.  Lengths, offsets and ids are read on the GPU only (no host
    synchronisation); lengths past what exists count as all of it.

    Head dims up to 128 (``NotImplementedError`` above), fp16 / bf16 / fp32.
    Returns O, or (O, LSE) with ``return_softmax_lse``; gradients of q, k, v and
    ``distance_slopes``, none in forward mode (``NotImplementedError``).  Forward and backward may be captured into a HIP graph;
    inputs that an eager graph of another stream still holds are refused there
    (``RuntimeError``).
    """
    check_qkv(q, k, v, "flash_attention_v100_scored")
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    scale = check_scale(scale, D)
    softcap = check_softcap(softcap, scale)
    slopes = prefix = lens = None
    if distance_slopes is not None:
        slopes = check_slopes(distance_slopes, B, H, q.device)
    if prefix_lengths is not None:
        prefix = _ops.optional_lengths(prefix_lengths, "prefix_lengths", B, q.device)
        if not causal:
            raise ValueError("prefix_lengths needs causal=True (without it every key is seen)")
    if key_lengths is not None:
        lens = _ops.optional_lengths(key_lengths, "key_lengths", B, q.device)
    offsets, offset0 = None, 0
    if isinstance(query_offsets, torch.Tensor):
        offsets = _ops.optional_lengths(query_offsets, "query_offsets", B, q.device)
    elif query_offsets is not None:
        offset0 = int(query_offsets)
        if abs(offset0) > 1 << 30:
            raise ValueError(f"query_offsets must be within +-2^30, got {query_offsets}")
    q_docs = k_docs = None
    if documents is not None:
        q_docs = _check_documents(documents, "documents", B, Sq, q.device)
        if key_documents is None and Sk != Sq:
            raise ValueError(f"documents of {Sq} queries and {Sk} keys: give key_documents too")
        k_docs = q_docs if key_documents is None else _check_documents(key_documents, "key_documents", B, Sk, q.device)
    elif key_documents is not None:
        raise ValueError("key_documents needs documents")
    if DebugConfig.CHECK_NUMERICAL_STABILITY:
        check_numerical_stability(q, k, v, None)
    if DebugConfig.VALIDATE_OUTPUTS:
        for t, name in ((q, "query"), (k, "key"), (v, "value"), (slopes, "distance_slopes")):
            check_tensor_nan_inf(t, name)
    rules = _ops.Rules(bool(causal), scale, softcap, slopes, prefix, lens, offsets, offset0, q_docs, k_docs)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (slopes is not None and slopes.requires_grad)):
        _ops.check_capture(q, k, v, slopes)
        out = ScoredAttentionFunction.apply(q, k, v, slopes, rules, return_softmax_lse)
        o, lse = out if return_softmax_lse else (out, None)
    else:
        o, lse, _ = _ops.scored_fwd(q, k, v, rules, return_softmax_lse)
    if DebugConfig.VALIDATE_OUTPUTS:
        check_tensor_nan_inf(o, "output")
    return (o, lse) if return_softmax_lse else o
