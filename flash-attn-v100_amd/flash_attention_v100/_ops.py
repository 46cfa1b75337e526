"""Binding of the operators around attention (C ABI ``include/fa_ops.h``) of the
gfx950 kernel library: attention with scored rules, new tokens after a shared
prefix, rotary positions.  Same library, host module, status codes and errors as
:mod:`._lib`; nothing is kept between calls and there is no fallback."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib

OPS_VERSION = 2
MAX_HEAD_DIM = 128

_I64x2, _I64x3, _I64x4 = ctypes.c_int64 * 2, ctypes.c_int64 * 3, ctypes.c_int64 * 4
_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class ScoredArgs(ctypes.Structure):
    _fields_ = (
        [(n, _P) for n in ("q", "k", "v", "o", "lse", "dout", "dq", "dk", "dv", "dslopes")]
        + [(n + "_stride", _I64x4) for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv")]
        + [(n, _I32) for n in ("batch", "seqlen_q", "seqlen_k", "num_heads", "num_heads_kv", "head_dim", "dtype",
                               "causal")]
        + [("scale", _F), ("softcap", _F), ("slopes", _P), ("slopes_batch_stride", _I64), ("prefix_lengths", _P),
           ("key_lengths", _P), ("query_offsets", _P), ("query_offset", _I32), ("q_documents", _P),
           ("k_documents", _P), ("q_documents_stride", _I64), ("k_documents_stride", _I64), ("lse_near", _P)])


class PrefixArgs(ctypes.Structure):
    _fields_ = (
        [(n, _P) for n in ("q", "k_prefix", "v_prefix", "k", "v", "o", "lse")]
        + [("q_stride", _I64x4), ("kp_stride", _I64x3), ("vp_stride", _I64x3), ("k_stride", _I64x4),
           ("v_stride", _I64x4), ("o_stride", _I64x4)]
        + [(n, _I32) for n in ("batch", "seqlen_q", "prefix_len", "seqlen_k", "num_heads", "num_heads_kv", "head_dim",
                               "dtype")]
        + [("scale", _F), ("softcap", _F), ("slopes", _P), ("slopes_batch_stride", _I64), ("key_lengths", _P)])


class RotaryArgs(ctypes.Structure):
    _fields_ = (
        [(n, _P) for n in ("q", "q_out", "k", "k_out")]
        + [(n + "_stride", _I64x4) for n in ("q", "q_out", "k", "k_out")]
        + [("table", _P), ("positions", _P), ("positions_stride", _I64x2), ("table_positions", _I64)]
        + [(n, _I32) for n in ("positions_64", "batch", "seqlen", "num_heads", "num_heads_k", "head_dim", "rotary_dim",
                               "dtype", "interleaved", "inverse")])


EXPORTS = ("fa_ops_version", "fa_scored_check", "fa_scored_fwd_workspace_size", "fa_scored_bwd_workspace_size",
           "fa_scored_fwd", "fa_scored_bwd", "fa_prefix_check", "fa_prefix_workspace_size", "fa_prefix_fwd",
           "fa_rotary_table", "fa_rotary_check", "fa_rotary")

ROTARY_SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3}

_ops_lib = None
_ops_host = None


def load() -> ctypes.CDLL:
    """The kernel library with the operators' functions typed."""
    global _ops_lib
    if _ops_lib is not None:
        return _ops_lib
    lib = _lib.load()
    missing = [n for n in EXPORTS if not hasattr(lib, n)]
    if missing:
        raise _lib.FlashAttentionExtensionError(f"{_lib.LIB_PATH} has no {', '.join(missing)}; build it with "
                                                "`python flash-attn-v100_amd/build.py`")
    ptr, size = ctypes.POINTER, ctypes.c_size_t
    for name, res, args in (
            ("fa_ops_version", _I32, []),
            ("fa_scored_check", _I32, [ptr(ScoredArgs), _I32]),
            ("fa_scored_fwd_workspace_size", size, [ptr(ScoredArgs)]),
            ("fa_scored_bwd_workspace_size", size, [ptr(ScoredArgs)]),
            ("fa_scored_fwd", _I32, [ptr(ScoredArgs), _P, size, _P]),
            ("fa_scored_bwd", _I32, [ptr(ScoredArgs), _P, size, _P]),
            ("fa_prefix_check", _I32, [ptr(PrefixArgs)]),
            ("fa_prefix_workspace_size", size, [ptr(PrefixArgs)]),
            ("fa_prefix_fwd", _I32, [ptr(PrefixArgs), _P, size, _P]),
            ("fa_rotary_table", _I32, [_P, _I64, _I32, _I32] + [ctypes.c_double] * 6 + [_P]),
            ("fa_rotary_check", _I32, [ptr(RotaryArgs)]),
            ("fa_rotary", _I32, [ptr(RotaryArgs), _P])):
        f = getattr(lib, name)
        f.restype, f.argtypes = res, args
    v = lib.fa_ops_version()
    if v != OPS_VERSION:
        raise _lib.FlashAttentionExtensionError(f"{_lib.LIB_PATH} has operator version {v}, expected {OPS_VERSION}")
    _ops_lib = lib
    return lib


def host():
    """The host module, its operators bound (once) to the library."""
    global _ops_host
    if _ops_host is not None:
        return _ops_host
    lib, mod = load(), _lib._host()
    if not hasattr(mod, "bind_ops"):
        raise _lib.FlashAttentionExtensionError(f"{_lib.HOST_PATH} has no operators; build both with "
                                                "`python flash-attn-v100_amd/build.py`")
    addr = [ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.fa_ops_version, lib.fa_scored_fwd_workspace_size, lib.fa_scored_fwd, lib.fa_scored_bwd_workspace_size,
        lib.fa_scored_bwd, lib.fa_prefix_workspace_size, lib.fa_prefix_fwd, lib.fa_rotary)]
    try:
        mod.bind_ops(addr[0], ctypes.sizeof(ScoredArgs), ctypes.sizeof(PrefixArgs), ctypes.sizeof(RotaryArgs), *addr[1:])
    except RuntimeError as e:
        raise _lib.FlashAttentionExtensionError(f"{_lib.HOST_PATH}: {e}; build both with "
                                                "`python flash-attn-v100_amd/build.py`") from e
    _ops_host = mod
    return mod


def padded(d: int, dtype: torch.dtype) -> int:
    """The head dim with its rows filled to whole 16-byte chunks: zero columns
    change no score and give zero columns of the outputs, which are dropped."""
    n = 4 if dtype == torch.float32 else 8
    return -(-d // n) * n


class Rules(NamedTuple):
    """The rules of a scored attention call, in the order the host module takes them."""

    causal: bool
    scale: float
    softcap: float
    slopes: Optional[torch.Tensor]
    prefix: Optional[torch.Tensor]
    lens: Optional[torch.Tensor]
    offsets: Optional[torch.Tensor]
    offset0: int
    q_docs: Optional[torch.Tensor]
    k_docs: Optional[torch.Tensor]


def scored_fwd(q, k, v, rules: Rules, want_lse: bool = True, for_backward: bool = False):
    """(o, lse or None, lse_near or None) of ``fa_scored_fwd``; checked tensors.
    ``for_backward`` (with ``want_lse``): lse_near where ``scored_bwd`` needs it."""
    D = q.shape[-1]
    dp = padded(D, q.dtype)
    if dp != D:
        q, k, v = (_lib._pad_d(t, dp) for t in (q, k, v))
    st, o, lse, near = host().scored_fwd(q, k, v, *rules, want_lse, for_backward, _lib._raw_stream(q))
    if st:
        _lib._check("fa_scored_fwd", st)
    return _lib._unpad_d(o, D), lse, near


def scored_bwd(q, k, v, o, do, lse, near, rules: Rules, want_dslopes: bool):
    """(dq, dk, dv, dslopes or None) of ``fa_scored_bwd``."""
    D = q.shape[-1]
    dp = padded(D, q.dtype)
    if dp != D:
        q, k, v, o, do = (_lib._pad_d(t, dp) for t in (q, k, v, o, do))
    st, dq, dk, dv, ds = host().scored_bwd(q, k, v, o, do, lse, near, *rules, want_dslopes, _lib._raw_stream(q))
    if st:
        _lib._check("fa_scored_bwd", st)
    if dp != D:
        dq, dk, dv = (_lib._unpad_d(t, D) for t in (dq, dk, dv))
    return dq, dk, dv, ds


def prefix_fwd(q, k_prefix, v_prefix, k, v, scale, softcap, slopes, lens, want_lse):
    """(o, lse or None) of ``fa_prefix_fwd``."""
    D = q.shape[-1]
    dp = padded(D, q.dtype)
    if dp != D:
        q, k_prefix, v_prefix, k, v = (_lib._pad_d(t, dp) for t in (q, k_prefix, v_prefix, k, v))
    st, o, lse = host().prefix_fwd(q, k_prefix, v_prefix, k, v, scale, softcap, slopes, lens, want_lse,
                                   _lib._raw_stream(q))
    if st:
        _lib._check("fa_prefix_fwd", st)
    return _lib._unpad_d(o, D), lse


def rotary(q, k, table, positions, interleaved, inverse, inplace):
    """(q', k' or None) of ``fa_rotary``."""
    st, qo, ko = host().rotary(q, k, table, positions, interleaved, inverse, inplace, _lib._raw_stream(q))
    if st:
        _lib._check("fa_rotary", st)
    return qo, ko


def rotary_table(positions: int, rotary_dim: int, scaling: int, base: float, factor: float, original: float, low: float,
                 high: float, mul: float, device) -> torch.Tensor:
    table = torch.empty((positions, rotary_dim), device=device, dtype=torch.float32)
    with torch.cuda.device(table.device):
        st = load().fa_rotary_table(table.data_ptr() if positions else None, positions, rotary_dim, scaling, base, factor,
                                    original, low, high, mul, _lib._stream(table))
    if st:
        _lib._check("fa_rotary_table", st)
    return table


def check_dual(what: str, *inputs) -> None:
    """Refuses inputs of forward-mode differentiation: their tangents would be lost."""
    if host().dual(*inputs):
        raise NotImplementedError(f"{what} has no forward-mode derivative (torch.autograd.forward_ad)")


def check_capture(*inputs) -> None:
    """Refuses a call to be differentiated inside a stream capture on an input
    whose gradient would leave the capture: one whose node another stream made, as
    a leaf's accumulator that an eager graph keeps alive.  The backward would make
    that stream wait on the capture, which ends the process at the capture's end."""
    if torch.cuda.is_current_stream_capturing() and host().on_other_stream(*inputs):
        raise RuntimeError("captured backward: an input belongs to an autograd graph of another stream that is still "
                           "alive; drop that graph's outputs before the capture, or capture on detached inputs")


def optional_lengths(t: Optional[torch.Tensor], name: str, B: int, device) -> Optional[torch.Tensor]:
    """An optional (B,) integer tensor on the inputs' device."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if tuple(t.shape) != (B,):
        raise ValueError(f"{name} must have shape {(B,)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t
