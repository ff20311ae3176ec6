"""Attention of new tokens over a paged key/value cache, and the writes that fill and compact the cache.

The serving side of the framework's attention (the reference has no counterpart): decoding of single tokens, chunks of a
prompt, and verification of a tree of drafted tokens, with the sliding window and sinks of ``window_attn_fwd`` or all of
the context visible.

The cache is a pair of pools ``[num_pages, Hkv, page_size, D]``.  ``page_table`` (int32 ``[B, max_pages]``) names the
pages of each sequence in order; entries outside the pool (-1, say) are pages the sequence does not have.
``cache_lens`` (int32 ``[B]``) counts a sequence's tokens *with* the ``T`` new ones, whose keys and values
``cache_append`` has put at positions ``cache_lens[b] - T .. cache_lens[b] - 1``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _cabi
from .bsa_attn_interface import _ceil_div
from .window_attn import _MAX_LEN, _check_lens, _check_qkv, _check_scale, _check_window, _launch_window_fwd, _out_buffers

_c_i64x3 = _cabi._c_i64x3

__all__ = ["cached_attn_fwd", "tree_mask_from_parents", "cache_append", "cache_keep"]

MAX_TREE_TOKENS = 64


def _check_cache(k_cache, v_cache, page_table, cache_lens, B: int, device):
    for t in (k_cache, v_cache):
        assert t.dim() == 4 and t.device == device, "the pools must be [num_pages, Hkv, page_size, D] on the device of q"
        # a pool is never copied: its rows have to be addressable as they lie
        st = t.stride()
        assert (st[3] == 1 and t.data_ptr() % 16 == 0 and st[0] > 0 and st[1] > 0 and st[2] > 0
                and (st[0] | st[1] | st[2]) % 8 == 0), (
            "the pools must have unit last stride, 16-byte aligned rows and no broadcast dimension")
    assert k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype, "K and V pools must match"
    num_pages, Hkv, page_size, D = k_cache.shape
    assert num_pages >= 1 and Hkv >= 1 and page_size >= 1, "the pools hold no page"
    assert page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.shape[0] == B, (
        f"page_table must be int32 of shape ({B}, max_pages)")
    assert page_table.device == device and page_table.shape[1] * page_size <= _MAX_LEN
    cache_lens = _check_lens(cache_lens, B, device, "cache_lens")
    assert cache_lens is not None, "cache_lens must be given"
    return page_table.contiguous(), cache_lens


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
    ``cache_lens[b] - T + (number of its bits) - 1``; window and sinks go by these positions.  An entry 0 is an unused slot.

    Rows that see nothing give ``out = 0`` and ``lse = -inf``: unused slots, tokens at negative positions
    (``cache_lens[b] < T``), sequences without pages.  Tokens whose page is not in the pool are not visible.  What the
    pages hold behind ``cache_lens[b]`` is never used.  The call is inference only: it has no gradient.
    """
    window, sink_tokens = _check_window(_MAX_LEN if window is None else window, sink_tokens)
    _check_qkv(q, k_cache, v_cache, layout)
    shape = q.shape
    B, Hq, T, D = shape if layout == "bhsd" else (shape[0], shape[2], shape[1], shape[3])
    page_table, cache_lens = _check_cache(k_cache, v_cache, page_table, cache_lens, B, q.device)
    Hkv, page_size = k_cache.shape[1], k_cache.shape[2]
    assert k_cache.shape[3] == D and Hq % Hkv == 0, "the pools must match q's head dimension, and Hkv divide Hq"
    assert page_size in (16, 32, 64) or page_size % 128 == 0, (
        f"page_size must be 16, 32, 64 or a multiple of 128, got {page_size}")
    scale = _check_scale(softmax_scale, D)
    if tree_mask is not None:
        assert T <= MAX_TREE_TOKENS, f"a tree has at most {MAX_TREE_TOKENS} drafts, got {T}"
        assert tree_mask.dtype == torch.int64 and tree_mask.shape == (B, T) and tree_mask.device == q.device, (
            f"tree_mask must be int64 of shape ({B}, {T}) on the device of q")
        tree_mask = tree_mask.contiguous()
    assert T <= _MAX_LEN
    out, lse_buf = _out_buffers(q, out, lse, return_lse or lse is not None, B, Hq, T)
    if out.numel() == 0 or page_table.shape[1] == 0:
        out.zero_()
        if lse_buf is not None:
            lse_buf.fill_(float("-inf"))
        return out, lse_buf
    G = Hq // Hkv
    pack = 1 < G <= 128
    capacity = page_table.shape[1] * page_size
    span = min(T, 128) + min(window, capacity)
    key_tiles, in_window = _ceil_div(capacity, 128), _ceil_div(span, 128) + 2
    ragged = key_tiles <= in_window  # the lists are as long as the sequences, not as the window
    key_tiles = min(key_tiles, in_window)
    _launch_window_fwd(q, k_cache, v_cache, out, lse_buf, layout, (B, Hq, Hkv, T, 0, D), kv_lens=cache_lens,
                       window=window, sinks=sink_tokens, scale=scale, pack_gqa=pack, key_tiles=key_tiles, ragged=ragged,
                       page_table=page_table, tree_mask=tree_mask, page_size=page_size)
    return out, lse_buf


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


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, cache_lens: torch.Tensor, *, layout: str = "bhsd"
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Writes the keys and values of ``T`` new tokens (``[B, Hkv, T, D]``, ``layout="bshd"``: ``[B, T, Hkv, D]``) of every
    sequence at positions ``cache_lens[b] - T .. cache_lens[b] - 1``, in place; returns the pools.

    Tokens at negative positions and tokens whose page is not in the pool are dropped; nothing else is touched.  A page
    must not be reached through two sequences' tables for writing.  BF16 or FP16, ``D`` a multiple of 8, any page size.
    """
    assert layout in ("bhsd", "bshd"), f"layout must be 'bhsd' or 'bshd', got {layout!r}"
    assert k.dim() == 4 and k.shape == v.shape and k.is_cuda and v.device == k.device, "k and v must match, on CUDA"
    assert k.dtype == v.dtype == k_cache.dtype and k.dtype in (torch.float16, torch.bfloat16), (
        "k, v and the pools must all be float16 or all bfloat16")
    shape = k.shape
    B, H, T, D = shape if layout == "bhsd" else (shape[0], shape[2], shape[1], shape[3])
    page_table, cache_lens = _check_cache(k_cache, v_cache, page_table, cache_lens, B, k.device)
    num_pages, pool_heads, page_size, pool_dim = k_cache.shape
    assert pool_heads == H and pool_dim == D and D % 8 == 0, "the pools must match k's heads and head dimension"
    if B == 0 or T == 0 or page_table.shape[1] == 0:
        return k_cache, v_cache

    def rows(t):
        st = t.stride()
        if st[3] != 1 or t.data_ptr() % 16 != 0 or (st[0] | st[1] | st[2]) % 8 != 0:
            t = t.clone(memory_format=torch.contiguous_format)
            st = t.stride()
        return t, _c_i64x3(st[0], st[1], st[2]) if layout == "bhsd" else _c_i64x3(st[0], st[2], st[1])

    (k_k, k_st), (v_k, v_st) = rows(k), rows(v)
    _cabi.launch(_cabi.load().bsa_cache_append, "bsa_cache_append", k.device, k_k.data_ptr(), v_k.data_ptr(),
                 k_cache.data_ptr(), v_cache.data_ptr(), k_st, v_st, _cabi.strides3(k_cache), _cabi.strides3(v_cache),
                 page_table.data_ptr(), cache_lens.data_ptr(), B, H, T, D, page_table.shape[1], page_size, num_pages)
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
    assert k_cache.is_cuda and k_cache.dtype in (torch.float16, torch.bfloat16), "the pools must be float16 or bfloat16 on CUDA"
    assert isinstance(num_drafts, int) and not isinstance(num_drafts, bool) and num_drafts >= 1, "num_drafts must be an int >= 1"
    B = cache_lens.shape[0]
    device = k_cache.device
    page_table, cache_lens = _check_cache(k_cache, v_cache, page_table, cache_lens, B, device)
    assert k_cache.shape[3] % 8 == 0, "the head dimension must be a multiple of 8"
    assert path.dtype == torch.int32 and path.dim() == 2 and path.shape[0] == B and path.device == device, (
        f"path must be int32 of shape ({B}, n) on the device of the pools")
    path, path_lens = path.contiguous(), _check_lens(path_lens, B, device, "path_lens")
    assert path_lens is not None, "path_lens must be given"
    if B == 0:
        return cache_lens.clone()
    if path.shape[1] == 0 or page_table.shape[1] == 0:
        path = torch.full((B, 1), -1, dtype=torch.int32, device=device)
    if page_table.shape[1] == 0:
        page_table = torch.full((B, 1), -1, dtype=torch.int32, device=device)
    new_lens = torch.empty_like(cache_lens)
    num_pages, H, page_size, D = k_cache.shape
    _cabi.launch(_cabi.load().bsa_cache_keep, "bsa_cache_keep", device, k_cache.data_ptr(), v_cache.data_ptr(),
                 _cabi.strides3(k_cache), _cabi.strides3(v_cache), page_table.data_ptr(), cache_lens.data_ptr(),
                 path.data_ptr(), path_lens.data_ptr(), new_lens.data_ptr(), B, H, num_drafts, path.shape[1], D,
                 page_table.shape[1], page_size, num_pages)
    return new_lens
