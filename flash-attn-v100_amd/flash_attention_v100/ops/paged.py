"""Attention of new tokens, or of a tree of drafted tokens, over a cache whose keys
lie in pages.  Forward only (serving).

The N new tokens of a sequence are the last of its ``key_lengths[b]`` filled ones:
their keys and values are in the cache (:func:`paged_cache_write_v100`).  For token
i and key j of sequence b and head h::

    x = scale * q_i . k_j
    s = softcap * tanh(x / softcap)  (x without a cap)
        - distance_slopes[h] * (tokens from j to i on the way that i sees)

and O is the softmax of s over the keys that i sees, times V: every key up to its
own place or, with ``parents``, the tokens before the N new ones, those on its way
through the tree and itself.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _ops, _paged
from ..config import DebugConfig
from ..utils import check_tensor_nan_inf
from .scored import check_scale, check_slopes, check_softcap


WHAT = "flash_attention_v100_paged"


def _check_inputs(q, k_cache, v_cache, key_lengths, page_table) -> None:
    """Raises for what the attention does not take."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    if q.dim() != 4:
        raise ValueError("q must be 4-dimensional [batch, tokens, num_heads, head_dim]")
    _paged.check_cache(WHAT, k_cache, v_cache, page_table, key_lengths, q.shape[0], False)
    if q.dtype != k_cache.dtype or q.device != k_cache.device or k_cache.shape[3] != q.shape[3]:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} does not match k_cache {tuple(k_cache.shape)} {k_cache.dtype}, or "
                         "its device")
    if q.shape[2] == 0 or q.shape[2] % k_cache.shape[2]:
        raise ValueError(f"num_heads {q.shape[2]} must be a positive multiple of num_heads_kv {k_cache.shape[2]}")
    _ops.check_dual(WHAT, q)
    if torch.is_grad_enabled() and q.requires_grad:
        raise NotImplementedError(f"{WHAT} has no backward: call it under torch.no_grad()")


def flash_attention_v100_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_lengths: Optional[torch.Tensor] = None,
    page_table: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    *,
    parents: Optional[torch.Tensor] = None,
    softcap: Optional[float] = None,
    distance_slopes: Optional[torch.Tensor] = None,
    return_softmax_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of q (B, N, H, D), the newest N tokens of each sequence, over a
    cache; the formula is in the module docstring.

    ``k_cache``, ``v_cache``: (pages, page_size, Hkv, D) with ``page_table`` (B, M):
    token x of sequence b lies in row ``x % page_size`` of page
    ``page_table[b, x // page_size]``; page_size is a multiple of 16.  A number that
    is no page holds no keys.  Without a table (B, S, Hkv, D): a row of tokens a
    sequence.  They are read as they are, never copied.
    ``key_lengths``: (B,) filled tokens, the new ones among them; all there is room
    for without it, and where they are more than that (M pages, or S).  Token i lies at place ``key_lengths[b] - N + i``; at a negative
    one (a free slot of the batch has length 0) it sees nothing: zero output, LSE
    -inf.
    ``parents``: (N,) or (B, N): the token that each one follows, an index below its
    own, or -1 behind the tokens before the new ones; anything else is padding, and
    so is what follows padding: it sees nothing and is seen by none.  N is at most
    256 then (``NotImplementedError`` above).
    ``softcap`` and ``distance_slopes`` as in :func:`flash_attention_v100_scored`;
    distances are counted along the tree.
    Tables, lengths and trees are int32 or int64 (converted at each call), read on
    the GPU only.  What lies in places that a token does not see does not reach it,
    infinities and NaN neither.

    Head dims up to 128 whose rows are whole 16-byte chunks, fp16 / bf16 / fp32.
    Inputs that require grad are refused while grad mode is on
    (``NotImplementedError``).
    """
    if not _paged.host().paged_ok(q, k_cache, v_cache, key_lengths, page_table):
        _check_inputs(q, k_cache, v_cache, key_lengths, page_table)
    B, N, H, D = q.shape
    scale = check_scale(scale, D)
    softcap = check_softcap(softcap, scale)
    slopes = None if distance_slopes is None else check_slopes(distance_slopes, B, H, q.device)
    if parents is not None:
        _paged.check_ints(parents, "parents", ((N,), (B, N)), q.device)
        if N > _paged.MAX_TREE_NODES:
            raise NotImplementedError(f"a tree has at most {_paged.MAX_TREE_NODES} tokens, got {N}")
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{WHAT} has no backward: call it under torch.no_grad()")
    o, lse = _paged.paged_fwd(q, k_cache, v_cache, key_lengths, page_table, parents, slopes, scale, softcap,
                              return_softmax_lse)
    if DebugConfig.VALIDATE_OUTPUTS:
        check_tensor_nan_inf(o, "output")
    return (o, lse) if return_softmax_lse else o
