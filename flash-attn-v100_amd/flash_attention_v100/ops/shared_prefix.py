"""New tokens of a batch of sequences that share a long prefix (a system prompt,
a document asked about many times): the prefix's keys and values are held and
read once for the whole batch.  Forward only (serving)."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _ops
from ..config import DebugConfig
from ..utils import check_numerical_stability, check_tensor_nan_inf
from .scored import check_qkv, check_scale, check_slopes, check_softcap


def flash_attention_v100_shared_prefix(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    key_lengths: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    *,
    softcap: Optional[float] = None,
    distance_slopes: Optional[torch.Tensor] = None,
    return_softmax_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of q (B, Sq, H, D), the newest Sq tokens of each sequence, over
    ``k_prefix``, ``v_prefix`` (P, Hkv, D), shared by the batch, followed by each
    sequence's own k, v (B, Sk, Hkv, D), of which the first ``key_lengths[b]``
    are filled (all without it; the new tokens are the last of them).

    Query i of sequence b stands at own position ``key_lengths[b] - Sq + i``: it
    sees the whole prefix and its own keys up to that position; at a negative one
    (a free slot of the batch has length 0) it sees nothing: zero output, LSE
    -inf.  ``softcap`` and ``distance_slopes`` as in
    :func:`flash_attention_v100_scored`, distances counted through the prefix.
    Equal to attention over the concatenated keys up to the order of float32
    sums.  Inputs that require grad are refused while grad mode is on
    (``NotImplementedError``).
    """
    check_qkv(q, k, v, "flash_attention_v100_shared_prefix")
    B, Sq, H, D = q.shape
    for t in (k_prefix, v_prefix):
        if not isinstance(t, torch.Tensor):
            raise TypeError("k_prefix, v_prefix must be torch.Tensor instances")
        if t.dim() != 3 or tuple(t.shape[1:]) != tuple(k.shape[2:]) or t.shape != k_prefix.shape:
            raise ValueError(f"k_prefix, v_prefix must have shape (P, {k.shape[2]}, {D}), got {tuple(k_prefix.shape)}, "
                             f"{tuple(v_prefix.shape) if isinstance(v_prefix, torch.Tensor) else v_prefix}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError("k_prefix, v_prefix must have the dtype and device of q")
    _ops.check_dual("flash_attention_v100_shared_prefix", k_prefix, v_prefix)
    scale = check_scale(scale, D)
    softcap = check_softcap(softcap, scale)
    slopes = check_slopes(distance_slopes, B, H, q.device)
    lens = _ops.optional_lengths(key_lengths, "key_lengths", B, q.device)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (q, k_prefix, v_prefix, k, v, slopes)):
        raise NotImplementedError("flash_attention_v100_shared_prefix has no backward: call it under torch.no_grad()")
    if DebugConfig.CHECK_NUMERICAL_STABILITY:
        check_numerical_stability(q, k, v, None)
    o, lse = _ops.prefix_fwd(q, k_prefix, v_prefix, k, v, scale, softcap, slopes, lens, return_softmax_lse)
    if DebugConfig.VALIDATE_OUTPUTS:
        check_tensor_nan_inf(o, "output")
    return (o, lse) if return_softmax_lse else o
