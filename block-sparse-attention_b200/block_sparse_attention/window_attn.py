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
from .bsa_attn_interface import _ceil_div, _tma_ready, maybe_contiguous

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


def _addressable(t: torch.Tensor) -> torch.Tensor:
    """``_tma_ready``, and a copy also of contiguous tensors that start between two 16-byte boundaries."""
    r = _tma_ready(t, 2)
    return r if r.data_ptr() % 16 == 0 else _tma_ready(t.clone(memory_format=torch.contiguous_format), 2)


def _can_hold(t: torch.Tensor) -> bool:
    """Whether the kernels can write rows of this BHSD view with 16-byte stores."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(t.shape[d] == 1 or (t.stride(d) > 0 and t.stride(d) % 8 == 0) for d in range(3)))


def _window_splits(items: int, key_tiles: int, num_sms: int) -> int:
    """Number of parts the key tiles of a query tile are dealt to.  Two CTAs fit an SM; when the query tiles alone fill
    less than half of those places, each is split as often as the places (and its key tiles) allow.  Splitting costs a
    second launch and fp32 partial rows, so a grid that is half full already stays unsplit."""
    places = 2 * num_sms
    if items < 1 or 2 * items > places:
        return 1
    return max(1, min(places // items, key_tiles, 256))


def _launch_window_fwd(*, q, k, v, out, lse, kv_lens, window, sinks, scale, page_table=None, tree_mask=None,
                       pack_gqa=False, page_size=0, key_tiles=1):
    """q, out are BHSD views; k, v BHSD views or (with a page table) [pages, H, page_size, D] pools."""
    lib = _cabi.load()
    device = q.device
    B, Hq, Sq, D = q.shape
    Hkv = k.shape[1]
    q_k, k_k, v_k = _addressable(q), _addressable(k), _addressable(v)
    out_k = out if _can_hold(out) else torch.empty(out.shape, dtype=out.dtype, device=device)
    out_view = _tma_ready(out_k, 2)
    lse_k = lse
    if lse is not None and not lse.is_contiguous():
        lse_k = torch.empty(lse.shape, dtype=torch.float32, device=device)

    G = Hq // Hkv
    tiles = _ceil_div(Sq, 128 // G) * Hkv if pack_gqa else _ceil_div(Sq, 128) * Hq
    splits = _window_splits(B * tiles, key_tiles, int(lib.bsa_num_sms(device.index or 0)))
    args = _cabi.WindowFwdArgs()
    args.q, args.k, args.v = q_k.data_ptr(), k_k.data_ptr(), v_k.data_ptr()
    args.out, args.lse = out_view.data_ptr(), _cabi.ptr(lse_k)
    args.kv_lens, args.page_table, args.tree_mask = _cabi.ptr(kv_lens), _cabi.ptr(page_table), _cabi.ptr(tree_mask)
    partial_o = partial_lse = None
    if splits > 1:
        partial_o = torch.empty((splits, B, Hq, Sq, D), dtype=torch.float32, device=device)
        partial_lse = torch.empty((splits, B, Hq, Sq), dtype=torch.float32, device=device)
        args.partial_o, args.partial_lse = partial_o.data_ptr(), partial_lse.data_ptr()
    args.status = _cabi.status_buffer(device).data_ptr()
    args.q_stride, args.k_stride, args.v_stride = _cabi.strides3(q_k), _cabi.strides3(k_k), _cabi.strides3(v_k)
    args.o_stride = _cabi.strides3(out_view)
    args.dtype = _dtype_code(q.dtype)
    args.B, args.Hq, args.Hkv, args.Sq, args.Sk, args.D = B, Hq, Hkv, Sq, (0 if page_size else k.shape[2]), D
    args.window, args.sinks = window, sinks
    if page_table is not None:
        args.max_pages, args.page_size, args.num_pages = page_table.shape[1], page_size, k.shape[0]
    args.pack_gqa = 1 if pack_gqa else 0
    args.splits = splits
    args.softmax_scale = scale
    with torch.cuda.device(device):
        _cabi.check(lib.bsa_window_fwd(args, _cabi.stream_ptr(device)), "bsa_window_fwd")
    if out_k is not out:
        out.copy_(out_k)
    if lse is not None and lse_k is not lse:
        lse.copy_(lse_k)


def _out_buffers(q, out, lse, want_lse, B, H, S):
    device = q.device
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
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
    assert q.dim() == 4 and k.dim() == 4 and v.dim() == 4
    assert q.is_cuda and k.is_cuda and v.is_cuda, "inputs must be on CUDA device"
    assert q.device == k.device == v.device, "Q/K/V must be on the same CUDA device"
    assert q.dtype == k.dtype == v.dtype, "inputs must have the same dtype"
    assert q.dtype in (torch.float16, torch.bfloat16), "inputs must be float16 or bfloat16"
    assert q.shape[-1] in (64, 96, 128), f"head dimension must be 64, 96 or 128, got {q.shape[-1]}"


def _views(layout, *tensors):
    return [t if layout == "bhsd" else t.transpose(1, 2) for t in tensors]


def _check_shapes(qb, kb, vb):
    B, Hq, Sq, D = qb.shape
    Bk, Hkv, Sk, Dk = kb.shape
    assert vb.shape == kb.shape and Bk == B and Dk == D, "K and V must match Q's batch and head dimension, and each other"
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
    q, k, v = [maybe_contiguous(t) for t in (q, k, v)]
    qb, kb, vb = _views(layout, q, k, v)
    B, Hq, Hkv, Sq, Sk, D = _check_shapes(qb, kb, vb)
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
    _launch_window_fwd(q=qb, k=kb, v=vb, out=_views(layout, out)[0], lse=lse_buf, kv_lens=kv_lens, window=window,
                       sinks=sink_tokens, scale=scale, pack_gqa=pack, key_tiles=key_tiles)
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
    q, k, v, out, dout = [maybe_contiguous(t) for t in (q, k, v, out, dout)]
    assert out.dtype == dout.dtype == q.dtype and lse.dtype == torch.float32
    assert all(t.device == q.device for t in (out, dout, lse)), "all tensors must be on the device of q"
    assert out.shape == q.shape and dout.shape == q.shape
    qb, kb, vb, ob, dob = _views(layout, q, k, v, out, dout)
    B, Hq, Hkv, Sq, Sk, D = _check_shapes(qb, kb, vb)
    assert lse.shape == (B, Hq, Sq)
    device = q.device
    kv_lens = _check_lens(kv_lens, B, device, "kv_lens")
    scale = _check_scale(softmax_scale, D)

    def _grad(buf, like):
        if buf is None:
            return torch.empty(like.shape, dtype=like.dtype, device=device)
        assert buf.shape == like.shape and buf.dtype == like.dtype and buf.device == device
        return buf

    grads = [_grad(dq, q), _grad(dk, k), _grad(dv, v)]
    if q.numel() == 0 or k.numel() == 0:
        for g in grads:
            g.zero_()
        return tuple(grads)
    lib = _cabi.load()
    held = [g if _can_hold(g) else torch.empty(g.shape, dtype=g.dtype, device=device) for g in _views(layout, *grads)]
    held = [_tma_ready(h, 2) for h in held]
    views = [_addressable(t) for t in (dob, qb, kb, vb, ob)]
    lse_c = lse.contiguous()
    ws_bytes = int(lib.bsa_window_bwd_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, window, sink_tokens))
    workspace = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=device)
    a = _cabi.WindowBwdArgs()
    a.dout, a.q, a.k, a.v, a.out = (t.data_ptr() for t in views)
    a.lse = lse_c.data_ptr()
    a.dq, a.dk, a.dv = (t.data_ptr() for t in held)
    a.kv_lens = _cabi.ptr(kv_lens)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    a.status = _cabi.status_buffer(device).data_ptr()
    a.do_stride, a.q_stride, a.k_stride, a.v_stride, a.o_stride = (_cabi.strides3(t) for t in views)
    a.dq_stride, a.dk_stride, a.dv_stride = (_cabi.strides3(t) for t in held)
    a.dtype = _dtype_code(q.dtype)
    a.B, a.Hq, a.Hkv, a.Sq, a.Sk, a.D = B, Hq, Hkv, Sq, Sk, D
    a.window, a.sinks = window, sink_tokens
    a.softmax_scale = scale
    with torch.cuda.device(device):
        _cabi.check(lib.bsa_window_bwd(a, _cabi.stream_ptr(device)), "bsa_window_bwd")
    for g, h in zip(_views(layout, *grads), held):
        if h.data_ptr() != g.data_ptr():
            g.copy_(h)
    return tuple(grads)


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
