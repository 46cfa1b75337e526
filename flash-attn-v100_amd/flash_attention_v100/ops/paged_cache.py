"""The cache that :func:`flash_attention_v100_paged` reads: rows of new tokens written,
drafted tokens accepted, sequences forked and freed, pages moved together.

A cache is a pool of pages, ``k_cache`` and ``v_cache`` (pages, page_size, Hkv, D), or
(layers, pages, page_size, Hkv, D) where one table serves several layers, with a
``page_table`` (B, M) and ``key_lengths`` (B,).  A page is in use while it is among
the first ``ceil(key_lengths[b] / page_size)`` columns of a sequence: freeing one is
setting its length to 0.  A length counts as 0 where it is negative, and as the room, M
pages, where it is more: a sequence that is told to grow past it stays full, and the new
tokens that are written take its last places, over the rows that were there (a caller that
may reach the end asks :func:`paged_cache_fork_v100` for room, which has none to give, or
counts).  Everything is read and decided on the GPU (no host
synchronisation), and every call may be captured into a HIP graph.  A number that is
no page holds nothing: nothing is written to it or moved from it.  k_cache and v_cache,
which every operator here writes, must not share memory (``ValueError``).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _ops, _paged


def paged_cache_write_v100(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_lengths: Optional[torch.Tensor] = None,
    page_table: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Writes k, v (B, N, Hkv, D), the newest N tokens of each sequence, into the cache:
    token i at place ``key_lengths[b] - N + i`` (the lengths count them, up to the room), a
    negative place is left out.  With a leading dimension of layers on the cache, k and v have
    it too.  Without ``page_table`` the cache is (B, S, Hkv, D), a row of tokens a
    sequence.  Returns (k_cache, v_cache), which are written in place; two sequences
    that share a page must not write the same place of it.  k and v must not lie in the
    caches' memory (``ValueError``).
    """
    if not _paged.host().write_ok(k, v, k_cache, v_cache, key_lengths, page_table):
        _check_write(k, v, k_cache, v_cache, key_lengths, page_table)
    _paged.cache_write(k, v, k_cache, v_cache, key_lengths, page_table)
    return k_cache, v_cache


def _check_write(k, v, k_cache, v_cache, key_lengths, page_table) -> None:
    what = "paged_cache_write_v100"
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dim() not in (4, 5):
            raise ValueError(f"{name} must be [batch, tokens, num_heads_kv, head_dim], or that with a leading dimension of "
                             "layers")
    _paged.check_cache(what, k_cache, v_cache, page_table, key_lengths, k.shape[-4], True)
    if k.shape != v.shape or k.dim() != k_cache.dim() or k.shape[-2:] != k_cache.shape[-2:] or (
            k.dim() == 5 and k.shape[0] != k_cache.shape[0]):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match the cache {tuple(k_cache.shape)}")
    for name, t in (("k", k), ("v", v)):
        if t.dtype != k_cache.dtype or t.device != k_cache.device:
            raise ValueError(f"{name} must have the dtype and device of the cache")
        if any(_paged.host().shares(t, x) for x in (k_cache, v_cache)):
            raise ValueError(f"{name} must not lie in the cache's memory")
    _ops.check_dual(what, k, v)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
        raise NotImplementedError(f"{what} has no backward: call it under torch.no_grad()")


def paged_cache_accept_v100(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_lengths: Optional[torch.Tensor],
    path: torch.Tensor,
    drafted: int,
    page_table: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Of the ``drafted`` newest tokens of each sequence keeps those of ``path`` (B, A):
    ascending indices among them, ended by the first entry that is not above the one
    before it or not below ``drafted`` (-1 behind the last).  Their rows move together,
    in every layer and in place.  Returns the new key lengths (B,), int32:
    ``key_lengths[b] - drafted`` and the number kept.  A sequence of fewer than
    ``drafted`` tokens stays as it is.  The drafted tokens' pages must not be shared
    with another sequence.
    """
    if not _paged.host().accept_ok(k_cache, v_cache, path, key_lengths, page_table):
        _check_accept(k_cache, v_cache, key_lengths, path, page_table)
    drafted = int(drafted)
    if drafted < 0 or drafted >= 1 << 31:
        raise ValueError(f"drafted must not be negative, got {drafted}")
    return _paged.cache_accept(k_cache, v_cache, path, key_lengths, page_table, drafted)


def _check_accept(k_cache, v_cache, key_lengths, path, page_table) -> None:
    what = "paged_cache_accept_v100"
    if not isinstance(path, torch.Tensor):
        raise TypeError("path must be a torch.Tensor")
    if path.dim() != 2:
        raise ValueError(f"path must be 2-dimensional [batch, tokens], got shape {tuple(path.shape)}")
    _paged.check_cache(what, k_cache, v_cache, page_table, key_lengths, path.shape[0], True)
    _paged.check_ints(path, "path", (tuple(path.shape),), k_cache.device)


def paged_cache_fork_v100(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    key_lengths: Optional[torch.Tensor],
    sources: torch.Tensor,
    new_tokens: Union[int, torch.Tensor] = 0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """A new batch whose sequence b continues sequence ``sources[b]`` of this one: in
    several copies, once, or not at all (which frees its pages); -1, or any other
    number that is no sequence, makes an empty one.  It has room for ``new_tokens``
    more (an int, or (B',) integers), which its length counts from now on.

    Whole pages are shared.  A partly filled last page stays with the first sequence
    that continues its own; each other one gets a page of its own, into which the
    filled rows are copied, in every layer.  New pages are the lowest ones that the
    new batch neither shares nor keeps, given in its order.  A sequence whose tokens do
    not fit the table's columns is dropped (length 0, no pages), and so are the first
    one that the free pages do not suffice for and those after it that need any.

    Returns (page_table (B', M), key_lengths (B',)), int32, -1 in columns without a
    page; the old ones are left as they are, and no longer valid once new tokens are
    written.  Pools of at most 2^20 pages (``NotImplementedError`` above).
    """
    if not _paged.host().fork_ok(k_cache, v_cache, page_table, sources, key_lengths, new_tokens):
        _check_fork(k_cache, v_cache, page_table, key_lengths, sources, new_tokens)
    if not isinstance(new_tokens, torch.Tensor):
        new_tokens = int(new_tokens)
        if new_tokens < 0 or new_tokens >= 1 << 31:
            raise ValueError(f"new_tokens must not be negative, got {new_tokens}")
    _check_pages("paged_cache_fork_v100", k_cache)
    return _paged.cache_fork(k_cache, v_cache, page_table, sources, key_lengths, new_tokens)


def _check_fork(k_cache, v_cache, page_table, key_lengths, sources, new_tokens) -> None:
    what = "paged_cache_fork_v100"
    if page_table is None:
        raise TypeError("page_table must be a torch.Tensor")
    _paged.check_cache(what, k_cache, v_cache, page_table, key_lengths, None, True)
    if not isinstance(sources, torch.Tensor):
        raise TypeError("sources must be a torch.Tensor")
    if sources.dim() != 1:
        raise ValueError(f"sources must be 1-dimensional, got shape {tuple(sources.shape)}")
    _paged.check_ints(sources, "sources", (tuple(sources.shape),), k_cache.device)
    if isinstance(new_tokens, torch.Tensor):
        _paged.check_ints(new_tokens, "new_tokens", (tuple(sources.shape),), k_cache.device)


def paged_cache_compact_v100(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    key_lengths: Optional[torch.Tensor],
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Moves the U pages in use to the front of the pool, in every layer and in place:
    the k-th lowest one from U on goes to the k-th lowest free one below U, the others
    stay.  Returns (page_table (B, M), U), int32 (U of shape ()), -1 in columns that no
    token needs; pages from U on are free.  Pools of at most 2^20 pages
    (``NotImplementedError`` above).
    """
    what = "paged_cache_compact_v100"
    if page_table is None:
        raise TypeError("page_table must be a torch.Tensor")
    _paged.check_cache(what, k_cache, v_cache, page_table, key_lengths, None, True)
    _check_pages(what, k_cache)
    return _paged.cache_compact(k_cache, v_cache, page_table, key_lengths)


def _check_pages(what: str, k_cache: torch.Tensor) -> None:
    if k_cache.shape[-4] > _paged.MAX_POOL_PAGES:
        raise NotImplementedError(f"{what} takes pools of at most {_paged.MAX_POOL_PAGES} pages, got {k_cache.shape[-4]}")
