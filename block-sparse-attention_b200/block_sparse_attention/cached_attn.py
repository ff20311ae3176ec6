"""Attention of new tokens over a paged key/value cache, and the writes that fill and compact the cache.

The serving side of the framework's attention (the reference has no counterpart): decoding of single tokens, chunks of a
prompt, and verification of a tree of drafted tokens, with the sliding window and sinks of ``window_attn_fwd`` or all of
the context visible.

The cache is a pair of pools ``[num_pages, Hkv, page_size, D]``.  ``page_table`` (int32 ``[B, max_pages]``) names the
pages of each sequence in order; entries outside the pool (-1, say) are pages the sequence does not have.
``cache_lens`` (int32 ``[B]``) counts a sequence's tokens *with* the ``T`` new ones, whose keys and values
``cache_append`` has put at positions ``cache_lens[b] - T .. cache_lens[b] - 1``.  A length beyond the table
(``max_pages * page_size``) counts as the table's in every call, a negative one as 0.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _cabi
from .bsa_attn_interface import _ceil_div
from .overlap import check_apart, pairs_apart, spread
from .window_attn import (_MAX_LEN, _Plan, _bhsd, _check_buffers, _check_lens, _check_qkv, _check_scale, _check_window, _copied,
                          _dense, _fits, _make_plan, _meta, _run_plan)

__all__ = ["cached_attn_fwd", "tree_mask_from_parents", "cache_append", "cache_keep"]

MAX_TREE_TOKENS = 64


def _check_cache(k_cache, v_cache, page_table, cache_lens, B: int, device) -> None:
    """Everything is a ``_meta``."""
    for t in (k_cache, v_cache):
        assert len(t[0]) == 4 and t[3] == device, "the pools must be [num_pages, Hkv, page_size, D] on the device of q"
        # a pool is never copied: its rows have to be addressable as they lie
        assert _fits(t[1]), "the pools must have unit last stride, 16-byte aligned rows and no broadcast dimension"
    assert k_cache[0] == v_cache[0] and k_cache[2] == v_cache[2], "K and V pools must match"
    num_pages, Hkv, page_size, _ = k_cache[0]
    assert num_pages >= 1 and Hkv >= 1 and page_size >= 1, "the pools hold no page"
    assert page_table[2] == torch.int32 and len(page_table[0]) == 2 and page_table[0][0] == B, (
        f"page_table must be int32 of shape ({B}, max_pages)")
    assert page_table[3] == device and page_table[0][1] * page_size <= _MAX_LEN
    assert cache_lens is not None, "cache_lens must be given"
    _check_lens(cache_lens, B, device, "cache_lens")


def _check_pool_address(*pools: int) -> None:
    assert (pools[0] | pools[1]) % 16 == 0, "the pools must be 16-byte aligned"


@functools.lru_cache(maxsize=256, typed=True)
def _cached_plan(q, k_cache, v_cache, table, lens, tree, out, lse, window, sinks, softmax_scale, layout, want_lse) -> _Plan:
    window, sinks = _check_window(_MAX_LEN if window is None else window, sinks)
    _check_qkv(q, k_cache, v_cache, layout)
    B, Hq, T, D = q[0] if layout == "bhsd" else (q[0][0], q[0][2], q[0][1], q[0][3])
    _check_cache(k_cache, v_cache, table, lens, B, q[3])
    _, Hkv, page_size, pool_dim = k_cache[0]
    assert pool_dim == D and Hq % Hkv == 0, "the pools must match q's head dimension, and Hkv divide Hq"
    assert page_size in (16, 32, 64) or page_size % 128 == 0, (
        f"page_size must be 16, 32, 64 or a multiple of 128, got {page_size}")
    if tree is not None:
        assert T <= MAX_TREE_TOKENS, f"a tree has at most {MAX_TREE_TOKENS} drafts, got {T}"
        assert tree[2] == torch.int64 and tree[0] == (B, T) and tree[3] == q[3], (
            f"tree_mask must be int64 of shape ({B}, {T}) on the device of q")
    assert T <= _MAX_LEN
    capacity = table[0][1] * page_size
    span = min(T, 128) + min(window, capacity)
    key_tiles, in_window = _ceil_div(capacity, 128), _ceil_div(span, 128) + 2
    # (within a window the lists of key tiles are about equal, otherwise as long as the sequences)
    return _make_plan(q, k_cache, v_cache, out, lse, lens, layout, (B, Hq, Hkv, T, 0, D), window=window, sinks=sinks,
                      scale=_check_scale(softmax_scale, D), pack_gqa=1 < Hq // Hkv <= 128, key_tiles=min(key_tiles, in_window),
                      ragged=key_tiles <= in_window, empty=table[0][1] == 0, want_lse=want_lse, table=table, tree=tree)


def cached_attn_fwd(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_lens: torch.Tensor,
    *,
    tree_mask: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sink_tokens: int = 0,
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    layout: str = "bhsd",
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of the ``T`` newest tokens of every sequence over its cached keys; returns ``(out, lse_or_None)``.

    ``q`` is ``[B, Hq, T, D]`` (``layout="bshd"``: ``[B, T, Hq, D]``), BF16 or FP16, ``D`` 64, 96 or 128, ``Hq`` a multiple of
    the pools' ``Hkv``; ``page_size`` 16, 32, 64 or a multiple of 128.  Without ``tree_mask`` the new tokens follow each
    other: token ``i`` is at position ``cache_lens[b] - T + i`` and sees what ``window_attn_fwd`` shows it (``window=None``:
    every earlier token).

    ``tree_mask`` (int64 ``[B, T]``, ``T <= 64``; see ``tree_mask_from_parents``) makes the new tokens drafts of a tree: bit
    ``u`` of entry ``t`` says that draft ``t`` sees draft ``u``.  A draft's position is that of its text,
    ``cache_lens[b] - T + (number of its bits) - 1``; window and sinks go by these positions (all bits count, also those of
    drafts that would lie before a sequence shorter than the tree).  An entry 0 is an unused slot.

    Rows that see nothing give ``out = 0`` and ``lse = -inf``: unused slots, tokens at negative positions
    (``cache_lens[b] < T``), sequences without pages.  Tokens whose page is not in the pool are not visible.  What the
    pages hold behind ``cache_lens[b]``, for unused slots and before every window reaches no result.  ``out`` may be q.  The
    call is inference only: it has no gradient.
    """
    want_lse = return_lse or lse is not None
    plan = _cached_plan(_meta(q), _meta(k_cache), _meta(v_cache), _meta(page_table), _meta(cache_lens), _meta(tree_mask),
                        _meta(out), _meta(lse), window, sink_tokens, None if softmax_scale is None else float(softmax_scale),
                        layout, want_lse)
    _check_pool_address(k_cache.data_ptr(), v_cache.data_ptr())
    if out is not None or lse is not None:
        _check_buffers(plan, out, lse, q, k_cache, v_cache, cache_lens, page_table, tree_mask)
    res = _run_plan(plan, q, k_cache, v_cache, out, lse, cache_lens, page_table, tree_mask) if plan.direct else None
    if res is not None:
        return res
    page_table, cache_lens = page_table.contiguous(), cache_lens.contiguous()
    tree_mask = None if tree_mask is None else tree_mask.contiguous()
    return _copied(lambda q, k, v: cached_attn_fwd(q, k, v, page_table, cache_lens, tree_mask=tree_mask, window=window,
                                                   sink_tokens=sink_tokens, softmax_scale=softmax_scale, return_lse=want_lse,
                                                   layout=layout),
                   q, k_cache, v_cache, out, lse, layout)


def tree_mask_from_parents(parents: torch.Tensor) -> torch.Tensor:
    """Ancestor masks of trees of drafts, for ``cached_attn_fwd``.

    ``parents`` (int32 ``[B, T]``, ``T <= 64``) names each draft's parent: an earlier draft of the same row, or -1 for the
    sequence's last token.  Returns int64 ``[B, T]``: bit ``u`` of entry ``t`` is set iff ``u`` is ``t`` or an ancestor of it.
    Any other value (-2, say) makes the draft and its descendants unused slots: mask 0.
    """
    assert parents.is_cuda and parents.dtype == torch.int32 and parents.dim() == 2, "parents must be int32 [B, T] on CUDA"
    B, T = parents.shape
    assert T <= MAX_TREE_TOKENS, f"a tree has at most {MAX_TREE_TOKENS} drafts, got {T}"
    parents = parents.contiguous()
    mask = torch.empty((B, T), dtype=torch.int64, device=parents.device)
    if mask.numel() == 0:
        return mask
    _cabi.launch(_cabi.load().bsa_tree_mask, "bsa_tree_mask", parents.device, parents.data_ptr(), B, T, mask.data_ptr())
    return mask


class _WritePlan(NamedTuple):
    """A checked write of the cache: everything but the addresses, kept as in ``window_attn._Plan``."""

    direct: bool
    empty: bool
    apart: tuple  # of overlap.check_apart: k_cache, v_cache, k, v
    args: bytes = b""  # CacheArgs without addresses


def _written_pools(k_cache, v_cache, k=None, v=None) -> tuple:
    """Pools that are written share no memory with each other nor with the rows that are written to them."""
    for t in (k_cache, v_cache):
        assert spread(*t[:2]), "a pool that is written must not overlap itself"
    return pairs_apart((("k_cache", k_cache), ("v_cache", v_cache)), (("k", k), ("v", v)))


@functools.lru_cache(maxsize=256, typed=True)
def _append_plan(k, v, k_cache, v_cache, table, lens, layout) -> _WritePlan:
    assert layout in ("bhsd", "bshd"), f"layout must be 'bhsd' or 'bshd', got {layout!r}"
    assert len(k[0]) == 4 and k[0] == v[0] and k[4] and v[3] == k[3], "k and v must match, on CUDA"
    assert k[2] == v[2] == k_cache[2] and k[2] in (torch.float16, torch.bfloat16), (
        "k, v and the pools must all be float16 or all bfloat16")
    B, H, T, D = k[0] if layout == "bhsd" else (k[0][0], k[0][2], k[0][1], k[0][3])
    _check_cache(k_cache, v_cache, table, lens, B, k[3])
    num_pages, pool_heads, page_size, pool_dim = k_cache[0]
    assert pool_heads == H and pool_dim == D and D % 8 == 0, "the pools must match k's heads and head dimension"
    apart = _written_pools(k_cache, v_cache, k, v)
    if B == 0 or T == 0 or table[0][1] == 0:
        return _WritePlan(True, True, apart)
    rows_ok = all(t[1][3] == 1 and (t[1][0] | t[1][1] | t[1][2]) % 8 == 0 for t in (k, v))
    if not (rows_ok and _dense(table) and _dense(lens)):
        return _WritePlan(False, False, apart)
    return _WritePlan(True, False, apart, bytes(_cabi.CacheArgs(
        *[None] * 9, _bhsd(k[1], layout), _bhsd(v[1], layout), k_cache[1][:3], v_cache[1][:3], B, H, T, D, table[0][1], page_size,
        num_pages, 0)))


@functools.lru_cache(maxsize=256, typed=True)
def _keep_plan(k_cache, v_cache, table, lens, path, path_lens, num_drafts) -> _WritePlan:
    assert k_cache[4] and k_cache[2] in (torch.float16, torch.bfloat16), "the pools must be float16 or bfloat16 on CUDA"
    assert isinstance(num_drafts, int) and not isinstance(num_drafts, bool) and num_drafts >= 1, "num_drafts must be an int >= 1"
    B, device = table[0][0], k_cache[3]
    _check_cache(k_cache, v_cache, table, lens, B, device)
    num_pages, H, page_size, D = k_cache[0]
    assert D % 8 == 0, "the head dimension must be a multiple of 8"
    assert path[2] == torch.int32 and len(path[0]) == 2 and path[0][0] == B and path[3] == device, (
        f"path must be int32 of shape ({B}, n) on the device of the pools")
    assert path_lens is not None, "path_lens must be given"
    _check_lens(path_lens, B, device, "path_lens")
    apart = _written_pools(k_cache, v_cache)
    if B == 0 or table[0][1] == 0:  # (a table without places holds no draft)
        return _WritePlan(True, True, apart)
    if path[0][1] == 0 or not all(_dense(t) for t in (table, lens, path, path_lens)):
        return _WritePlan(False, False, apart)
    return _WritePlan(True, False, apart, bytes(_cabi.CacheArgs(
        *[None] * 9, (0, 0, 0), (0, 0, 0), k_cache[1][:3], v_cache[1][:3], B, H, num_drafts, D, table[0][1], page_size, num_pages,
        path[0][1])))


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, cache_lens: torch.Tensor, *, layout: str = "bhsd"
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Writes the keys and values of ``T`` new tokens (``[B, Hkv, T, D]``, ``layout="bshd"``: ``[B, T, Hkv, D]``) of every
    sequence at positions ``cache_lens[b] - T .. cache_lens[b] - 1``, in place; returns the pools.

    Tokens at negative positions and tokens whose page is not in the pool are dropped; nothing else is touched.  A page
    must not be reached through two entries of the table for writing, and k and v share no memory with the pools.  BF16 or
    FP16, ``D`` a multiple of 8, any page size.
    """
    plan = _append_plan(_meta(k), _meta(v), _meta(k_cache), _meta(v_cache), _meta(page_table), _meta(cache_lens), layout)
    pools, at = (k_cache.data_ptr(), v_cache.data_ptr()), (k.data_ptr(), v.data_ptr())
    _check_pool_address(*pools)
    check_apart(plan.apart, pools + at)
    if plan.empty:
        return k_cache, v_cache
    if not plan.direct or (at[0] | at[1]) % 16 != 0:
        k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        return cache_append(k, v, k_cache, v_cache, page_table.contiguous(), cache_lens.contiguous(), layout=layout)
    a = _cabi.CacheArgs.from_buffer_copy(plan.args)
    a.k, a.v = at
    a.k_cache, a.v_cache = pools
    a.page_table, a.lens = page_table.data_ptr(), cache_lens.data_ptr()
    _cabi.launch(_cabi.load().bsa_cache_append, "bsa_cache_append", k.device, a)
    return k_cache, v_cache


def cache_keep(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, cache_lens: torch.Tensor,
               path: torch.Tensor, path_lens: torch.Tensor, num_drafts: int) -> torch.Tensor:
    """Keeps the accepted drafts of every sequence and drops the others; returns the new lengths (int32 ``[B]``).

    The last ``num_drafts`` tokens of each sequence are drafts.  ``path`` (int32 ``[B, n]``) holds the numbers of the
    accepted ones in ascending order, ``path_lens`` (int32 ``[B]``) how many there are.  Draft ``path[b, i]`` moves to
    position ``cache_lens[b] - num_drafts + i``, in place; the new length is ``cache_lens[b] - num_drafts`` plus the
    number kept.  A path ends early at an entry that is not ascending or not a draft.  A sequence with fewer than
    ``num_drafts`` tokens is left as it is.  A move from or to a page that is not in the pool is dropped.
    """
    plan = _keep_plan(_meta(k_cache), _meta(v_cache), _meta(page_table), _meta(cache_lens), _meta(path), _meta(path_lens), num_drafts)
    pools = k_cache.data_ptr(), v_cache.data_ptr()
    _check_pool_address(*pools)
    check_apart(plan.apart, pools)
    if plan.empty:
        return cache_lens.clone()
    if not plan.direct:
        if path.shape[1] == 0:
            path = path.new_full((path.shape[0], 1), -1)
        return cache_keep(k_cache, v_cache, page_table.contiguous(), cache_lens.contiguous(), path.contiguous(),
                          path_lens.contiguous(), num_drafts)
    new_lens = torch.empty_like(cache_lens)
    a = _cabi.CacheArgs.from_buffer_copy(plan.args)
    a.k_cache, a.v_cache = pools
    a.page_table, a.lens = page_table.data_ptr(), cache_lens.data_ptr()
    a.path, a.path_lens, a.new_lens = path.data_ptr(), path_lens.data_ptr(), new_lens.data_ptr()
    _cabi.launch(_cabi.load().bsa_cache_keep, "bsa_cache_keep", k_cache.device, a)
    return new_lens
