"""Rotary positions for q and k: a table of cosines and sines, and the rotation.

Column pair j of the first R columns of a head turns by ``position * w_j``,
``w_j = base ** (-2 j / R)``; pairs are (j, j + R / 2) or, interleaved,
(2 j, 2 j + 1), and columns past R stay.  For contexts longer than a model was
trained on the angles may be scaled (:func:`rotary_table_v100`).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import _ops

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def rotary_table_v100(
    max_positions: int,
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: str = "none",
    factor: float = 1.0,
    original_positions: Optional[int] = None,
    low_rotations: float = 1.0,
    high_rotations: float = 32.0,
    attention_factor: Optional[float] = None,
    device: Union[str, torch.device, None] = None,
) -> torch.Tensor:
    """float32 table (max_positions, rotary_dim): row n holds cos(n w_j), then
    sin(n w_j) of the rotary_dim / 2 pairs, from angles in 64 bits.

    ``scaling``, by ``factor``: "none"; "linear": every w_j divided by it;
    "base": the base grows by factor ** (R / (R - 2)), which stretches the slowest
    pair by the factor and keeps the fastest; "ramp": pairs that turn at least
    ``high_rotations`` times over ``original_positions`` keep their w_j, those of
    at most ``low_rotations`` are divided, blended in between, and cosines and
    sines are multiplied by ``attention_factor`` (0.1 ln factor + 1 unless given;
    1 for the other scalings).  The blend is linear in the rotations; a model that
    blends over the pairs' index brings a table of its own, of the same layout."""
    if scaling not in _ops.ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {tuple(_ops.ROTARY_SCALINGS)}, got {scaling!r}")
    if not isinstance(max_positions, int) or max_positions < 1 or max_positions > 1 << 31:
        raise ValueError(f"max_positions must be a positive int, got {max_positions!r}")
    if not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 256:
        raise ValueError(f"rotary_dim must be even, 2..256, got {rotary_dim!r}")
    if not (math.isfinite(base) and base > 0):
        raise ValueError(f"base must be finite and positive, got {base}")
    if not (math.isfinite(factor) and factor > 0):
        raise ValueError(f"factor must be finite and positive, got {factor}")
    if scaling == "ramp":
        if original_positions is None or original_positions < 1:
            raise ValueError("scaling='ramp' needs original_positions")
        if not (math.isfinite(low_rotations) and math.isfinite(high_rotations) and high_rotations > low_rotations):
            raise ValueError(f"high_rotations must exceed low_rotations, got {low_rotations}, {high_rotations}")
    if attention_factor is None:
        attention_factor = 0.1 * math.log(factor) + 1.0 if scaling == "ramp" else 1.0
    if not math.isfinite(attention_factor):
        raise ValueError(f"attention_factor must be finite, got {attention_factor}")
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError("rotary_table_v100 requires a GPU device (there is no CPU path)")
    return _ops.rotary_table(max_positions, rotary_dim, _ops.ROTARY_SCALINGS[scaling], float(base), float(factor),
                             float(original_positions or 1), float(low_rotations), float(high_rotations),
                             float(attention_factor), dev)


class RotaryFunction(torch.autograd.Function):
    """Rotation and, backward, the transposed rotation of the gradients."""

    @staticmethod
    def forward(ctx, q, k, table, positions, interleaved):
        ctx.save_for_backward(table, positions)
        ctx.interleaved = interleaved
        qo, ko = _ops.rotary(q, k, table, positions, interleaved, False, False)
        return (qo, ko) if k is not None else qo

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        table, positions = ctx.saved_tensors
        need = ctx.needs_input_grad
        if need[0] and dk is not None and need[1]:
            gq, gk = _ops.rotary(dq, dk, table, positions, ctx.interleaved, True, False)
            return gq, gk, None, None, None
        gq = _ops.rotary(dq, None, table, positions, ctx.interleaved, True, False)[0] if need[0] else None
        gk = (_ops.rotary(dk, None, table, positions, ctx.interleaved, True, False)[0]
              if dk is not None and need[1] else None)
        return gq, gk, None, None, None


def _overlaps(shape, strides) -> bool:
    """Whether two indices of a tensor may share an element (strides checked from
    the smallest up; a negative answer is exact for views of dense tensors)."""
    end = 0
    for st, n in sorted((st, n) for st, n in zip(strides, shape) if n > 1):
        if st <= end:
            return True
        end += st * (n - 1)
    return False


def _disjoint(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether q and k share no element: different storages or address ranges, or
    heads of one packed tensor."""
    if q.numel() == 0 or k.numel() == 0 or q.untyped_storage().data_ptr() != k.untyped_storage().data_ptr():
        return True
    (q0, q1), (k0, k1) = ((t.storage_offset(), t.storage_offset() + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))
                          for t in (q, k))
    if q1 < k0 or k1 < q0:
        return True
    sh = q.stride(2) if q.shape[2] > 1 else k.stride(2) if k.shape[2] > 1 else abs(k0 - q0)
    gap = abs(k0 - q0)
    first, last = (q, k) if q0 < k0 else (k, q)
    if sh == 0 or gap % sh or gap // sh < first.shape[2] or any(
            t.shape[2] > 1 and t.stride(2) != sh for t in (q, k)) or any(
            q.shape[d] > 1 and q.stride(d) != k.stride(d) for d in (0, 1)):
        return False
    return not _overlaps((*first.shape[:2], gap // sh + last.shape[2], first.shape[3]), (*first.stride()[:2], sh, 1))


def _check_inputs(q, k, table, positions):
    """Raises for what the rotation does not take; positions as (B, S)."""
    _ops.check_dual("rotary_embedding_v100", q, k, table)
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dim() != 4:
            raise ValueError("Input tensors must be 4-dimensional [batch, seq_len, num_heads, head_dim]")
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.float32:
        raise ValueError("table must be a float32 (positions, rotary_dim) tensor (rotary_table_v100)")
    B, S, H, D = q.shape
    R = table.shape[1]
    if q.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"dtype must be one of {SUPPORTED_DTYPES}, got {q.dtype}")
    if k is not None and (k.dtype != q.dtype or k.device != q.device or k.shape[:2] != q.shape[:2] or k.shape[3] != D):
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} does not match q {tuple(q.shape)} {q.dtype}")
    if H == 0 or (k is not None and k.shape[2] == 0):
        raise ValueError("q and k need at least one head")
    if q.device.type != "cuda" or table.device != q.device:
        raise ValueError("rotary_embedding_v100 requires q, k and table on the same GPU device (there is no CPU path)")
    if D > 256:
        raise NotImplementedError(f"head_dim {D} has no kernel (1..256)")
    if R < 2 or R % 2 or R > D or table.shape[0] == 0:
        raise ValueError(f"table {tuple(table.shape)} does not fit head_dim {D}")
    if table.requires_grad:
        raise ValueError("the table has no gradient")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be an int32 or int64 tensor")
        if tuple(positions.shape) not in ((S,), (1, S), (B, S)):
            raise ValueError(f"positions must have shape {(S,)} or {(B, S)}, got {tuple(positions.shape)}")
        if positions.device != q.device:
            raise ValueError(f"positions must be on {q.device}, got {positions.device}")
        positions = positions.expand(B, S)
    return positions


def rotary_embedding_v100(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    table: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    *,
    interleaved: bool = False,
    inplace: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q (B, S, H, D) and k (B, S, Hkv, D) with their first ``table.shape[1]``
    columns rotated: (q', k'), or q' alone for ``k`` None; in one launch.

    ``table`` from :func:`rotary_table_v100`.  ``positions``: int32 or int64
    (B, S) or (S,), 0 .. S - 1 by default; read on the GPU only: a token at a
    negative position is left as it is, one at a position past the table becomes
    NaN.  ``inplace`` writes into q and k and returns them (refused for inputs
    that require grad while grad mode is on, and for inputs whose elements
    overlap).  Differentiable in q and k, not in forward mode
    (``NotImplementedError``).
    """
    if not _ops.host().rotary_ok(q, k, table, positions):
        positions = _check_inputs(q, k, table, positions)
    grad = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    if inplace:
        if grad:
            raise ValueError("inplace=True on inputs that require grad: call it under torch.no_grad()")
        for name, t in (("q", q), ("k", k)):
            if t is not None and ((t.shape[3] > 1 and t.stride(3) != 1) or _overlaps(t.shape, t.stride())):
                raise ValueError(f"inplace=True needs a {name} with unit column stride and no overlapping elements")
        if k is not None and not _disjoint(q, k):
            raise ValueError("inplace=True needs a q and k that share no element")
        return _pair(*_ops.rotary(q, k, table, positions, bool(interleaved), False, True))
    if grad:
        _ops.check_capture(q, k)
        return RotaryFunction.apply(q, k, table, positions, bool(interleaved))
    return _pair(*_ops.rotary(q, k, table, positions, bool(interleaved), False, False))


def _pair(q, k):
    return q if k is None else (q, k)
