"""Binding of the paged key/value cache (C ABI ``include/fa_paged.h``) of the gfx950
kernel library.  Same library, host module, status codes and errors as
:mod:`._lib`; nothing is kept between calls and there is no fallback."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib, _ops

PAGED_VERSION = 1
MAX_HEAD_DIM = 128
MAX_TREE_NODES = 256
MAX_POOL_PAGES = 1 << 20
PAGE_MULTIPLE = 16

_I64x4, _I64x5 = ctypes.c_int64 * 4, ctypes.c_int64 * 5
_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class PagePool(ctypes.Structure):
    _fields_ = (
        [("k", _P), ("v", _P), ("k_stride", _I64x5), ("v_stride", _I64x5)]
        + [(n, _I32) for n in ("layers", "pages", "page_size", "num_heads_kv", "head_dim", "dtype", "batch", "table_cols")]
        + [("page_table", _P), ("table_stride", _I64), ("key_lengths", _P)])


class PagedArgs(ctypes.Structure):
    _fields_ = [("pool", PagePool), ("q", _P), ("o", _P), ("lse", _P), ("q_stride", _I64x4), ("o_stride", _I64x4),
                ("seqlen_q", _I32), ("num_heads", _I32), ("scale", _F), ("softcap", _F), ("slopes", _P),
                ("slopes_batch_stride", _I64), ("parents", _P), ("parents_stride", _I64)]


class CacheWriteArgs(ctypes.Structure):
    _fields_ = [("pool", PagePool), ("k", _P), ("v", _P), ("k_stride", _I64x5), ("v_stride", _I64x5), ("tokens", _I32)]


class CacheAcceptArgs(ctypes.Structure):
    _fields_ = [("pool", PagePool), ("path", _P), ("path_stride", _I64), ("path_cols", _I32), ("tokens", _I32),
                ("new_lengths", _P)]


class CacheForkArgs(ctypes.Structure):
    _fields_ = [("pool", PagePool), ("sources", _P), ("more", _P), ("more_all", _I32), ("new_batch", _I32),
                ("new_table", _P), ("new_lengths", _P)]


class CacheCompactArgs(ctypes.Structure):
    _fields_ = [("pool", PagePool), ("new_table", _P), ("used", _P)]


STRUCTS = (PagedArgs, CacheWriteArgs, CacheAcceptArgs, CacheForkArgs, CacheCompactArgs)
EXPORTS = ("fa_paged_version", "fa_paged_check", "fa_paged_workspace_size", "fa_paged_fwd", "fa_cache_write_check",
           "fa_cache_write", "fa_cache_accept_check", "fa_cache_accept", "fa_cache_fork_check",
           "fa_cache_fork_workspace_size", "fa_cache_fork", "fa_cache_compact_check", "fa_cache_compact_workspace_size",
           "fa_cache_compact")

_paged_lib = None
_paged_host = None


def load() -> ctypes.CDLL:
    """The kernel library with the cache's functions typed."""
    global _paged_lib
    if _paged_lib is not None:
        return _paged_lib
    lib = _lib.load()
    missing = [n for n in EXPORTS if not hasattr(lib, n)]
    if missing:
        raise _lib.FlashAttentionExtensionError(f"{_lib.LIB_PATH} has no {', '.join(missing)}; build it with "
                                                "`python flash-attn-v100_amd/build.py`")
    ptr, size = ctypes.POINTER, ctypes.c_size_t
    lib.fa_paged_version.restype, lib.fa_paged_version.argtypes = _I32, []
    for name, args, ws in (("fa_paged", PagedArgs, True), ("fa_cache_write", CacheWriteArgs, False),
                           ("fa_cache_accept", CacheAcceptArgs, False), ("fa_cache_fork", CacheForkArgs, True),
                           ("fa_cache_compact", CacheCompactArgs, True)):
        run = getattr(lib, "fa_paged_fwd" if name == "fa_paged" else name)
        run.restype, run.argtypes = _I32, [ptr(args)] + ([_P, size, _P] if ws else [_P])
        check = getattr(lib, name + "_check")
        check.restype, check.argtypes = _I32, [ptr(args)]
        if ws:
            f = getattr(lib, name + "_workspace_size")
            f.restype, f.argtypes = size, [ptr(args)]
    v = lib.fa_paged_version()
    if v != PAGED_VERSION:
        raise _lib.FlashAttentionExtensionError(f"{_lib.LIB_PATH} has paged cache version {v}, expected {PAGED_VERSION}")
    _paged_lib = lib
    return lib


def host():
    """The host module, its cache operators bound (once) to the library."""
    global _paged_host
    if _paged_host is not None:
        return _paged_host
    lib, mod = load(), _lib._host()
    if not hasattr(mod, "bind_paged"):
        raise _lib.FlashAttentionExtensionError(f"{_lib.HOST_PATH} has no paged cache; build both with "
                                                "`python flash-attn-v100_amd/build.py`")
    addr = [ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.fa_paged_version, lib.fa_paged_workspace_size, lib.fa_paged_fwd, lib.fa_cache_write, lib.fa_cache_accept,
        lib.fa_cache_fork_workspace_size, lib.fa_cache_fork, lib.fa_cache_compact_workspace_size, lib.fa_cache_compact)]
    try:
        mod.bind_paged(addr[0], *(ctypes.sizeof(s) for s in STRUCTS), *addr[1:])
    except RuntimeError as e:
        raise _lib.FlashAttentionExtensionError(f"{_lib.HOST_PATH}: {e}; build both with "
                                                "`python flash-attn-v100_amd/build.py`") from e
    _paged_host = mod
    return mod


def paged_fwd(q, k_cache, v_cache, lens, table, parents, slopes, scale, softcap, want_lse):
    """(o, lse or None) of ``fa_paged_fwd``; checked tensors."""
    st, o, lse = host().paged_fwd(q, k_cache, v_cache, lens, table, parents, slopes, scale, softcap, want_lse,
                                  _lib._raw_stream(q))
    if st:
        _lib._check("fa_paged_fwd", st)
    return o, lse


def cache_write(k, v, k_cache, v_cache, lens, table) -> None:
    st = host().cache_write(k, v, k_cache, v_cache, lens, table, _lib._raw_stream(k_cache))
    if st:
        _lib._check("fa_cache_write", st)


def cache_accept(k_cache, v_cache, path, lens, table, tokens) -> torch.Tensor:
    st, new = host().cache_accept(k_cache, v_cache, path, lens, table, tokens, _lib._raw_stream(k_cache))
    if st:
        _lib._check("fa_cache_accept", st)
    return new


def cache_fork(k_cache, v_cache, table, sources, lens, more):
    st, table, lens = host().cache_fork(k_cache, v_cache, table, sources, lens, more, _lib._raw_stream(k_cache))
    if st:
        _lib._check("fa_cache_fork", st)
    return table, lens


def cache_compact(k_cache, v_cache, table, lens):
    st, table, used = host().cache_compact(k_cache, v_cache, table, lens, _lib._raw_stream(k_cache))
    if st:
        _lib._check("fa_cache_compact", st)
    return table, used


def check_ints(t, name: str, shapes, device) -> torch.Tensor:
    """An integer tensor of one of the shapes on the cache's device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} must have shape {' or '.join(str(s) for s in shapes)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t


def _overlaps(t: torch.Tensor) -> bool:
    """Whether two indices of a tensor may share an element (strides checked from the
    smallest up)."""
    end = 0
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st <= end:
            return True
        end += st * (n - 1)
    return False


def check_cache(what: str, k_cache, v_cache, table, lens, batch: Optional[int], written: bool) -> None:
    """Raises for a cache that the kernels do not take: pages (pages, page_size, Hkv, D),
    or (layers, ...) where ``written``, its page table and filled lengths.  ``batch``:
    that of the call (of the table where None)."""
    if host().pool_ok(k_cache, v_cache, table, lens, batch, written):
        return
    names = (("k_cache", k_cache), ("v_cache", v_cache))
    for name, t in names:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    _ops.check_dual(what, k_cache, v_cache)
    if k_cache.dim() != 4 and not (written and k_cache.dim() == 5):
        raise ValueError("k_cache, v_cache must be [pages, page_size, num_heads_kv, head_dim]"
                         + (", or that with a leading dimension of layers" if written else ""))
    if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype or v_cache.device != k_cache.device:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} {k_cache.dtype} and v_cache {tuple(v_cache.shape)} "
                         f"{v_cache.dtype} must match")
    if k_cache.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"dtype must be one of {tuple(_lib.DTYPE_CODES)}, got {k_cache.dtype}")
    if k_cache.device.type != "cuda":
        raise ValueError(f"{what} requires a cache on a GPU device (there is no CPU path)")
    pages, size, Hkv, D = k_cache.shape[-4:]
    es = k_cache.element_size()
    if D == 0 or D > MAX_HEAD_DIM or D * es % 16:
        raise NotImplementedError(f"{what} has no kernel for head_dim {D} of {k_cache.dtype} (up to {MAX_HEAD_DIM}, whole "
                                  "16-byte chunks)")
    if Hkv == 0 or (k_cache.dim() == 5 and k_cache.shape[0] == 0):
        raise ValueError("a cache needs a layer and a head")
    if torch.is_grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad):
        raise NotImplementedError(f"{what} has no backward: k_cache and v_cache must not require grad")
    for name, t in names:
        if t.stride(-1) != 1 or t.data_ptr() % 16 or any(st < 0 or st * es % 16 for st in t.stride()[:-1]):
            raise ValueError(f"{name} needs rows of unit stride that start at multiples of 16 bytes (it is not copied)")
        if written and _overlaps(t):
            raise ValueError(f"{name} has overlapping elements")
    if written and host().shares(k_cache, v_cache):
        raise ValueError("k_cache and v_cache must not lie in the same memory")
    if table is not None:
        if not isinstance(table, torch.Tensor):
            raise TypeError("page_table must be a torch.Tensor")
        if table.dim() != 2:
            raise ValueError(f"page_table must be 2-dimensional [batch, pages], got shape {tuple(table.shape)}")
        check_ints(table, "page_table", ((table.shape[0] if batch is None else batch, table.shape[1]),), k_cache.device)
        batch = table.shape[0]
        if size == 0 or size % PAGE_MULTIPLE:
            raise ValueError(f"a page must hold a multiple of {PAGE_MULTIPLE} tokens, got {size}")
    elif pages != batch:
        raise ValueError(f"without a page_table the cache has one row of tokens a sequence: {batch}, got {pages}")
    if lens is not None:
        check_ints(lens, "key_lengths", ((batch,),), k_cache.device)
