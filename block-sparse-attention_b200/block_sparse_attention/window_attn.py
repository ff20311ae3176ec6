"""Causal sliding-window attention with sink tokens: forward, backward and the autograd wrapper.

The companion of the block-sparse operators for models whose layers see a window of recent tokens and the first few
tokens of the sequence (the reference has no counterpart).  Tensor layouts, argument checks (``AssertionError``), the
handling of ``out`` / ``lse`` / gradient buffers and the return conventions are those of ``bsa_attn_fwd`` and
``bsa_attn_bwd``.

Query token ``i`` sits at position ``p = i + Sk - Sq``; key ``j`` is visible to it iff
``p < len``, ``j <= p`` and (``j > p - window`` or ``j < sink_tokens``), with ``len = kv_lens[b]`` or ``Sk``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _cabi
from .bsa_attn_interface import _ceil_div, _tma_ready

__all__ = ["window_attn_fwd", "window_attn_bwd", "window_attention", "WindowAttentionFunction"]

MAX_SINK_TOKENS = 128
_MAX_LEN = 1 << 29


def _check_window(window, sink_tokens) -> Tuple[int, int]:
    assert isinstance(window, int) and not isinstance(window, bool) and window >= 1, "window must be an int >= 1"
    assert isinstance(sink_tokens, int) and not isinstance(sink_tokens, bool) and 0 <= sink_tokens <= MAX_SINK_TOKENS, (
        f"sink_tokens must be an int in [0, {MAX_SINK_TOKENS}]")
    return min(window, _MAX_LEN), sink_tokens


def _check_scale(softmax_scale, D: int) -> float:
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    assert scale > 0 and math.isfinite(scale), "softmax_scale must be positive and finite"
    return scale


def _check_lens(lens, B: int, device, name: str) -> Optional[torch.Tensor]:
    if lens is None:
        return None
    assert lens.dtype == torch.int32 and lens.shape == (B,), f"{name} must be int32 of shape ({B},)"
    assert lens.device == device, f"{name} must be on the device of q"
    return lens.contiguous()


def _dtype_code(dtype) -> int:
    return _cabi.BSA_DTYPE_F16 if dtype == torch.float16 else _cabi.BSA_DTYPE_BF16


def _rows(t: torch.Tensor, layout: str):
    """(tensor, BHSD strides) the tensor maps can address; copies only views that they cannot."""
    st = t.stride()
    st = (st[0], st[1], st[2], st[3]) if layout == "bhsd" else (st[0], st[2], st[1], st[3])
    if st[3] == 1 and st[0] > 0 and st[1] > 0 and st[2] > 0 and (st[0] | st[1] | st[2]) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, st[:3]
    view = _tma_ready(t if layout == "bhsd" else t.transpose(1, 2), 2)
    if view.data_ptr() % 16 != 0:  # contiguous, but starting between two 16-byte boundaries
        view = _tma_ready(view.clone(memory_format=torch.contiguous_format), 2)
    return view, view.stride()[:3]


def _can_hold(t: torch.Tensor, st) -> bool:
    """Whether the kernels can write the rows of a buffer with 16-byte stores."""
    return (t.stride(3) == 1 and st[0] > 0 and st[1] > 0 and st[2] > 0 and (st[0] | st[1] | st[2]) % 8 == 0
            and t.data_ptr() % 16 == 0)


def _stream_ctas(items: int, key_tiles: int, ragged: bool, num_sms: int) -> int:
    """How the work of a call is dealt: 0 = whole query tiles in turn, otherwise the number of CTAs that share the list of
    all key tiles evenly.  Sharing costs a second launch and fp32 rows of the cut query tiles, so it is for query tiles
    that do not fill the two places of every SM, and for lists of unequal lengths that only the device knows while the
    places get less than eight query tiles each (they do not even out)."""
    places = 2 * num_sms
    if items >= (8 * places if ragged else places) or key_tiles <= 1 or items * (key_tiles + 1) >= 1 << 31:
        return 0
    return min(places, items * key_tiles)


def _launch_window_fwd(q, k, v, out, lse, layout, shape, *, kv_lens, window, sinks, scale, pack_gqa, key_tiles, ragged,
                       page_table=None, tree_mask=None, page_size=0):
    """``shape`` is (B, Hq, Hkv, Sq, Sk, D); with a page table, k and v are [pages, Hkv, page_size, D] pools."""
    lib = _cabi.load()
    device = q.device
    B, Hq, Hkv, Sq, Sk, D = shape
    kv_layout = layout if page_table is None else "bhsd"
    (q_k, q_st), (k_k, k_st), (v_k, v_st) = _rows(q, layout), _rows(k, kv_layout), _rows(v, kv_layout)
    out_k, o_st = out, out.stride()
    o_st = (o_st[0], o_st[1], o_st[2]) if layout == "bhsd" else (o_st[0], o_st[2], o_st[1])
    if not _can_hold(out, o_st):
        out_k = torch.empty((B, Hq, Sq, D), dtype=out.dtype, device=device)
        o_st = out_k.stride()[:3]
    lse_k = lse
    if lse is not None and not lse.is_contiguous():
        lse_k = torch.empty(lse.shape, dtype=torch.float32, device=device)

    per_tile = 128 // (Hq // Hkv) if pack_gqa else 128  # query tokens of a tile
    items = B * _ceil_div(Sq, per_tile) * (Hkv if pack_gqa else Hq)
    ctas = _stream_ctas(items, key_tiles, ragged, lib.bsa_num_sms(device.index))
    joins = partial_o = partial_lse = None
    lists = 1
    if ctas:
        tiles = _ceil_div(Sq, per_tile)
        if page_table is not None and 1 < tiles <= ctas:  # new tokens over a long past: nearly the same keys
            lists = tiles
            ctas -= ctas % lists
        rows = 2 * ctas * min(Sq, per_tile) * (Hq // Hkv if pack_gqa else 1)
        workspace = q.new_empty(4 * ctas + rows * (D + 1), dtype=torch.float32)
        joins = workspace.data_ptr()
        partial_o = joins + 16 * ctas
        partial_lse = partial_o + 4 * rows * D
    paged = page_table is not None
    args = _cabi.WindowFwdArgs(
        q_k.data_ptr(), k_k.data_ptr(), v_k.data_ptr(), out_k.data_ptr(), _cabi.ptr(lse_k), _cabi.ptr(kv_lens),
        _cabi.ptr(page_table), _cabi.ptr(tree_mask), partial_o, partial_lse, joins, _cabi.status_buffer(device).data_ptr(), q_st,
        k_st, v_st, o_st, _dtype_code(q.dtype), B, Hq, Hkv, Sq, Sk, D, window, sinks, page_table.shape[1] if paged else 0,
        page_size, k.shape[0] if paged else 0, 1 if pack_gqa else 0, ctas, lists, scale)
    _cabi.launch(lib.bsa_window_fwd, "bsa_window_fwd", device, args)
    if out_k is not out:
        (out if layout == "bhsd" else out.transpose(1, 2)).copy_(out_k)
    if lse is not None and lse_k is not lse:
        lse.copy_(lse_k)


def _out_buffers(q, out, lse, want_lse, B, H, S):
    device = q.device
    if out is None:
        out = torch.empty_like(q)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == device
        assert out.stride(-1) == 1
    if lse is None:
        lse = torch.empty((B, H, S), dtype=torch.float32, device=device) if want_lse else None
    else:
        assert lse.shape == (B, H, S) and lse.dtype == torch.float32 and lse.device == device
    return out, lse


def _check_qkv(q, k, v, layout):
    assert layout in ("bhsd", "bshd"), f"layout must be 'bhsd' or 'bshd', got {layout!r}"
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "inputs must be 4-D"
    assert q.is_cuda and k.is_cuda and v.is_cuda, "inputs must be on CUDA device"
    assert q.device == k.device == v.device, "Q/K/V must be on the same CUDA device"
    assert q.dtype == k.dtype == v.dtype, "inputs must have the same dtype"
    assert q.dtype in (torch.float16, torch.bfloat16), "inputs must be float16 or bfloat16"
    assert q.shape[-1] in (64, 96, 128), f"head dimension must be 64, 96 or 128, got {q.shape[-1]}"


def _check_shapes(q, k, v, layout):
    h, n = (1, 2) if layout == "bhsd" else (2, 1)
    qs, ks = q.shape, k.shape
    B, Hq, Sq, D, Hkv, Sk = qs[0], qs[h], qs[n], qs[3], ks[h], ks[n]
    assert v.shape == ks and ks[0] == B and ks[3] == D, "K and V must match Q's batch and head dimension, and each other"
    assert Hkv >= 1 and Hq % Hkv == 0, "the number of query heads must be a multiple of the number of KV heads"
    assert Sq <= _MAX_LEN and Sk <= _MAX_LEN
    return B, Hq, Hkv, Sq, Sk, D


def window_attn_fwd(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    window: int,
    sink_tokens: int = 0,
    *,
    kv_lens: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    layout: str = "bhsd",
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Sliding-window attention forward; always returns ``(out, lse_or_None)``.

    ``q`` is ``[B, Hq, Sq, D]``, ``k`` and ``v`` ``[B, Hkv, Sk, D]`` (``layout="bshd"``: heads and tokens swapped), BF16
    or FP16, ``D`` 64, 96 or 128, ``Hq`` a multiple of ``Hkv``; any strides whose last is 1.  A query sees the
    ``window`` newest keys up to itself and the first ``sink_tokens`` (at most 128) keys; ``Sq < Sk`` are the last
    ``Sq`` tokens of the sequence (a chunk of a prompt).  ``kv_lens`` (int32 ``[B]``) gives the tokens of each
    sequence of a padded batch: keys and queries at positions from ``kv_lens[b]`` on take no part, whatever they hold.
    Rows that see nothing give ``out = 0`` and ``lse = -inf``.  LSE (natural log, scale included, fp32 ``[B, Hq, Sq]``)
    is returned iff ``return_lse``, a gradient is required or an ``lse`` buffer was passed.

    Inside a sequence, a NaN or infinity in a value that some query sees may reach other queries of the same 128 keys.
    """
    window, sink_tokens = _check_window(window, sink_tokens)
    _check_qkv(q, k, v, layout)
    want_lse = return_lse or lse is not None or q.requires_grad or k.requires_grad or v.requires_grad
    shape = B, Hq, Hkv, Sq, Sk, D = _check_shapes(q, k, v, layout)
    kv_lens = _check_lens(kv_lens, B, q.device, "kv_lens")
    scale = _check_scale(softmax_scale, D)
    out, lse_buf = _out_buffers(q, out, lse, want_lse, B, Hq, Sq)
    if out.numel() == 0 or Sk == 0:
        out.zero_()
        if lse_buf is not None:
            lse_buf.fill_(-math.inf)
        return out, lse_buf
    # one head's queries do not fill a 128-row tile: tiles of several heads then, so that the group reads its keys once
    pack = Hq > Hkv and Sq < 128 and Hq // Hkv <= 128
    span = min(Sq, 128) + min(window, Sk)
    key_tiles = min(_ceil_div(Sk, 128), _ceil_div(span, 128) + 2)
    _launch_window_fwd(q, k, v, out, lse_buf, layout, shape, kv_lens=kv_lens, window=window, sinks=sink_tokens,
                       scale=scale, pack_gqa=pack, key_tiles=key_tiles, ragged=False)
    return out, lse_buf


def window_attn_bwd(
    dout: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    window: int,
    sink_tokens: int = 0,
    *,
    kv_lens: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    dq: Optional[torch.Tensor] = None,
    dk: Optional[torch.Tensor] = None,
    dv: Optional[torch.Tensor] = None,
    layout: str = "bhsd",
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward of ``window_attn_fwd``: returns ``(dq, dk, dv)`` in the shapes of q, k, v.

    The gradients of a KV head sum over the query heads that share it, in fp32 and in a fixed order, so repeated calls
    are bit-identical.  Tokens behind ``kv_lens`` get zero gradients.  ``out`` and ``lse`` are those of the forward call
    with the same arguments.
    """
    window, sink_tokens = _check_window(window, sink_tokens)
    _check_qkv(q, k, v, layout)
    assert out.dtype == dout.dtype == q.dtype and lse.dtype == torch.float32
    device = q.device
    assert out.device == dout.device == lse.device == device, "all tensors must be on the device of q"
    assert out.shape == q.shape and dout.shape == q.shape
    B, Hq, Hkv, Sq, Sk, D = _check_shapes(q, k, v, layout)
    assert lse.shape == (B, Hq, Sq)
    kv_lens = _check_lens(kv_lens, B, device, "kv_lens")
    scale = _check_scale(softmax_scale, D)

    def _grad(buf, like):
        if buf is None:
            return torch.empty_like(like)
        assert buf.shape == like.shape and buf.dtype == like.dtype and buf.device == device
        return buf

    grads = dq, dk, dv = _grad(dq, q), _grad(dk, k), _grad(dv, v)
    if q.numel() == 0 or k.numel() == 0:
        for g in grads:
            g.zero_()
        return grads
    lib = _cabi.load()
    held, held_st = [], []
    for g in grads:
        st = g.stride()
        st = (st[0], st[1], st[2]) if layout == "bhsd" else (st[0], st[2], st[1])
        if not _can_hold(g, st):
            g = torch.empty((B, g.shape[1], g.shape[2], D) if layout == "bhsd" else (B, g.shape[2], g.shape[1], D),
                            dtype=g.dtype, device=device)
            st = g.stride()[:3]
        held.append(g)
        held_st.append(st)
    (do_k, do_st), (q_k, q_st), (k_k, k_st), (v_k, v_st), (o_k, o_st) = (_rows(t, layout) for t in (dout, q, k, v, out))
    lse_c = lse.contiguous()
    ws_bytes = max(16, lib.bsa_window_bwd_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, window, sink_tokens))
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8)
    a = _cabi.WindowBwdArgs(
        do_k.data_ptr(), q_k.data_ptr(), k_k.data_ptr(), v_k.data_ptr(), o_k.data_ptr(), lse_c.data_ptr(),
        held[0].data_ptr(), held[1].data_ptr(), held[2].data_ptr(), _cabi.ptr(kv_lens), workspace.data_ptr(),
        _cabi.status_buffer(device).data_ptr(), ws_bytes, do_st, q_st, k_st, v_st, o_st, held_st[0], held_st[1], held_st[2],
        _dtype_code(q.dtype), B, Hq, Hkv, Sq, Sk, D, window, sink_tokens, scale)
    _cabi.launch(lib.bsa_window_bwd, "bsa_window_bwd", device, a)
    for g, t in zip(grads, held):
        if t is not g:
            (g if layout == "bhsd" else g.transpose(1, 2)).copy_(t)
    return grads


class WindowAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sink_tokens, kv_lens, softmax_scale, layout):
        out, lse = window_attn_fwd(q, k, v, window, sink_tokens, kv_lens=kv_lens, softmax_scale=softmax_scale,
                                   return_lse=True, layout=layout)
        ctx.save_for_backward(q, k, v, out, lse, kv_lens)
        ctx.how = (window, sink_tokens, softmax_scale, layout)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lens = ctx.saved_tensors
        window, sink_tokens, softmax_scale, layout = ctx.how
        dq, dk, dv = window_attn_bwd(dout, q, k, v, out, lse, window, sink_tokens, kv_lens=kv_lens,
                                     softmax_scale=softmax_scale, layout=layout)
        return dq, dk, dv, None, None, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sink_tokens: int = 0,
                     kv_lens: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                     layout: str = "bhsd") -> torch.Tensor:
    """Differentiable sliding-window attention with sinks (see ``window_attn_fwd`` for the arguments)."""
    return WindowAttentionFunction.apply(q, k, v, window, sink_tokens, kv_lens, softmax_scale, layout)
