"""Causal sliding-window attention with sink tokens: forward, backward and the autograd wrapper.

The companion of the block-sparse operators for models whose layers see a window of recent tokens and the first few
tokens of the sequence (the reference has no counterpart).  Tensor layouts, argument checks (``AssertionError``), the
handling of ``out`` / ``lse`` / gradient buffers and the return conventions are those of ``bsa_attn_fwd`` and
``bsa_attn_bwd``.

Query token ``i`` sits at position ``p = i + Sk - Sq``; key ``j`` is visible to it iff
``p < len``, ``j <= p`` and (``j > p - window`` or ``j < sink_tokens``), with ``len = kv_lens[b]`` or ``Sk``.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _cabi
from .bsa_attn_interface import _ceil_div, _tma_ready
from .overlap import check_apart, pairs_apart, spread

__all__ = ["window_attn_fwd", "window_attn_bwd", "window_attention", "WindowAttentionFunction"]

MAX_SINK_TOKENS = 128
MAX_TEAM = 8
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


def _meta(t: Optional[torch.Tensor]):
    """What the checks of a call look at (everything but the address): the key of its plan."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device, t.is_cuda)


def _check_lens(lens, B: int, device, name: str) -> None:
    """``lens`` is a ``_meta``."""
    assert lens[2] == torch.int32 and lens[0] == (B,), f"{name} must be int32 of shape ({B},)"
    assert lens[3] == device, f"{name} must be on the device of q"


def _dtype_code(dtype) -> int:
    return _cabi.BSA_DTYPE_F16 if dtype == torch.float16 else _cabi.BSA_DTYPE_BF16


def _dense(t) -> bool:
    """Whether a tensor (its ``_meta``) is contiguous; a dimension of size 1 may have any stride."""
    n = 1
    for size, st in zip(reversed(t[0]), reversed(t[1])):
        if size != 1 and st != n:
            return False
        n *= size
    return True


def _bhsd(st, layout: str):
    return (st[0], st[1], st[2]) if layout == "bhsd" else (st[0], st[2], st[1])


def _fits(st) -> bool:
    """Whether 16-byte accesses and tensor maps can address rows with these element strides (from an aligned address)."""
    return st[3] == 1 and st[0] > 0 and st[1] > 0 and st[2] > 0 and (st[0] | st[1] | st[2]) % 8 == 0


def _aligned(t: torch.Tensor, layout: str) -> torch.Tensor:
    """The tensor itself if the kernels can address it, otherwise a copy that they can."""
    if _fits(t.stride()) and t.data_ptr() % 16 == 0:
        return t
    bhsd = _tma_ready(t if layout == "bhsd" else t.transpose(1, 2), 2)
    if bhsd.data_ptr() % 16 != 0:  # contiguous, but starting between two 16-byte boundaries
        bhsd = _tma_ready(bhsd.clone(memory_format=torch.contiguous_format), 2)
    return bhsd if layout == "bhsd" else bhsd.transpose(1, 2)


def _deal_work(items: int, key_tiles: int, rows: int, ragged: bool, num_sms: int) -> Tuple[int, int]:
    """How the work of a call is dealt, as ``(ctas, team)``: ``(0, 1)`` whole query tiles in turn, ``(0, n)`` a cluster of n
    CTAs for each query tile, ``(ctas, 1)`` that many CTAs share the list of all key tiles evenly.

    The cheapest of the three in key tiles of the busiest place (two places for each SM; a key tile takes 1.5 us there, two at
    once 1.9).  The costs choose between the three and are no forecast of a call; they are from before whole query tiles were dealt
    to heads in turn, which made those 5 to 27 % faster.  A team adds its start and the join through shared memory; sharing a list adds the search for each CTA's run, a second
    launch, the fp32 rows of the cut query tiles that go through memory, and neighbours that share fewer loads.  The
    coefficients fit times over 1 to 256 query tiles of 1 to 128 rows, lists of 2 to 256 key tiles, one token of
    four heads per KV head: 8 query tiles of 8 key tiles take 17.2 us whole, 9.9 as teams, 11.7 shared, of 64 key tiles 101,
    20.5 and 23.0; 16 query tiles of 128 full rows and 128 key tiles 204, 44.7 and 37.2; 128 of 16 key tiles 34.2, 42.4
    and 46.7.

    Lists of unequal lengths that only the device knows (``ragged``) are taken as half full on average: that is what
    sharing makes of them, while several whole query tiles for each place even out by themselves (sequences of equally
    spread lengths, 8 KV heads: 128 of up to 4096 tokens 310 us whole, 266 shared; 256 of up to 2048 276 and 316)."""
    places = 2 * num_sms
    if items < 1 or items * (key_tiles + 1) >= 1 << 31:
        return 0, 1
    load = items / places
    whole = key_tiles * (min(math.ceil(load), 0.5 * load + 0.42 * math.sqrt(load)) if ragged and load > 1 else math.ceil(load))
    ctas = min(places, items * key_tiles)
    stream = (0.625 if ragged else 1.25) * max(1.0, key_tiles * load) + 4 + 0.07 * ctas / items + 0.02 * (ctas + items) * rows / 128
    team = min(MAX_TEAM, key_tiles, places // items)
    teams = _ceil_div(key_tiles, team) + 2 + 0.1 * rows / team + 0.01 * items if team >= 2 else math.inf
    if teams < min(whole, stream):
        return 0, team
    return (ctas, 1) if stream < whole else (0, 1)


class _Plan(NamedTuple):
    """A checked call: everything but the addresses.  Kept by the shapes, strides, types and options of the call (a
    decoding loop makes the same call every step; the checks cost more than its launch)."""

    direct: bool            # the kernels can address the tensors as they are, up to the alignment of the addresses
    empty: bool             # no key or no query: zeros, nothing to launch
    out_shape: tuple
    lse_shape: Optional[tuple]  # None: no LSE is returned
    args: bytes             # WindowFwdArgs without addresses
    workspace: int          # floats
    partial_o: int          # byte offsets in it
    partial_lse: int
    apart: tuple            # of overlap.check_apart: out, lse, q, k, v, lens, table, tree
    q_dense: bool = False   # contiguous: empty_like, the cheaper call, gives the same


def _check_qkv(q, k, v, layout):
    """``q, k, v`` are ``_meta``s."""
    assert layout in ("bhsd", "bshd"), f"layout must be 'bhsd' or 'bshd', got {layout!r}"
    assert len(q[0]) == 4 and len(k[0]) == 4 and len(v[0]) == 4, "inputs must be 4-D"
    assert q[4] and k[4] and v[4], "inputs must be on CUDA device"
    assert q[3] == k[3] == v[3], "Q/K/V must be on the same CUDA device"
    assert q[2] == k[2] == v[2], "inputs must have the same dtype"
    assert q[2] in (torch.float16, torch.bfloat16), "inputs must be float16 or bfloat16"
    assert q[0][3] in (64, 96, 128), f"head dimension must be 64, 96 or 128, got {q[0][3]}"


def _check_shapes(q, k, v, layout):
    h, n = (1, 2) if layout == "bhsd" else (2, 1)
    B, Hq, Sq, D, Hkv, Sk = q[0], q[h], q[n], q[3], k[h], k[n]
    assert v == k and k[0] == B and k[3] == D, "K and V must match Q's batch and head dimension, and each other"
    assert Hkv >= 1 and Hq % Hkv == 0, "the number of query heads must be a multiple of the number of KV heads"
    assert Sq <= _MAX_LEN and Sk <= _MAX_LEN
    return B, Hq, Hkv, Sq, Sk, D


def _make_plan(q, k, v, out, lse, lens, layout, shape, *, window, sinks, scale, pack_gqa, key_tiles, ragged, empty, want_lse,
               table=None, tree=None) -> _Plan:
    """The part that the two forward calls share; tensors are ``_meta``s, ``shape`` is (B, Hq, Hkv, Sq, Sk, D)."""
    B, Hq, Hkv, Sq, Sk, D = shape
    device = q[3]
    if out is not None:
        assert out[0] == q[0] and out[2] == q[2] and out[3] == device, "out must match q"
        assert out[1][3] == 1 and spread(*out[:2]), "out must have unit last stride and not overlap itself"
    if lse is not None:
        assert lse[0] == (B, Hq, Sq) and lse[2] == torch.float32 and lse[3] == device, f"lse must be float32 ({B}, {Hq}, {Sq})"
        assert spread(*lse[:2]), "lse must not overlap itself"
    lse_shape = (B, Hq, Sq) if want_lse else None
    apart = pairs_apart((("out", out), ("lse", lse)), (("q", q), ("k", k), ("v", v), ("lengths", lens), ("page_table", table),
                                                       ("tree_mask", tree)), (("out", "q"),))  # (a query tile is read first)
    if empty or Sq == 0 or B == 0 or Hq == 0:
        return _Plan(True, True, tuple(q[0]), lse_shape, b"", 0, 0, 0, apart)
    kv_layout = layout if table is None else "bhsd"
    out_st = out[1] if out is not None else ((Hq * Sq * D, Sq * D, D, 1) if layout == "bhsd" else (Hq * Sq * D, Hq * D, D, 1))
    direct = (_fits(q[1]) and _fits(k[1]) and _fits(v[1]) and _fits(out_st)
              and all(t is None or _dense(t) for t in (lse, lens, table, tree)))
    if not direct:
        return _Plan(False, False, tuple(q[0]), lse_shape, b"", 0, 0, 0, apart)
    per_tile = 128 // (Hq // Hkv) if pack_gqa else 128  # query tokens of a tile
    tiles = _ceil_div(Sq, per_tile)
    items = B * tiles * (Hkv if pack_gqa else Hq)
    slot_rows = (Hq // Hkv if pack_gqa else 1) * min(Sq, per_tile)
    ctas, team = _deal_work(items, key_tiles, slot_rows, ragged, _cabi.load().bsa_num_sms(device.index))
    lists = 1
    if table is not None and 1 < tiles <= ctas:  # new tokens over a long past: nearly the same keys
        lists = tiles
        ctas -= ctas % lists
    rows = 2 * ctas * slot_rows
    args = _cabi.WindowFwdArgs(
        None, None, None, None, None, None, None, None, None, None, None, None, _bhsd(q[1], layout), _bhsd(k[1], kv_layout),
        _bhsd(v[1], kv_layout), _bhsd(out_st, layout), _dtype_code(q[2]), B, Hq, Hkv, Sq, Sk, D, window, sinks,
        table[0][1] if table is not None else 0, k[0][2] if table is not None else 0, k[0][0] if table is not None else 0,
        1 if pack_gqa else 0, ctas, lists, team, scale)
    # workspace: the list of joins (four ints a CTA), the pieces' rows, their LSE
    return _Plan(True, False, tuple(q[0]), lse_shape, bytes(args), (4 * ctas + rows * (D + 1)) if ctas else 0, 16 * ctas,
                 16 * ctas + 4 * rows * D, apart, q[1] == ((n := q[0])[1] * n[2] * n[3], n[2] * n[3], n[3], 1))


def _run_plan(plan: _Plan, q, k, v, out, lse, lens, table, tree):
    """Launches a checked call; returns (out, lse), or None if some address is not aligned (nothing was launched)."""
    if out is None:
        out = torch.empty_like(q) if plan.q_dense else q.new_empty(plan.out_shape)
    if lse is None and plan.lse_shape is not None:
        lse = q.new_empty(plan.lse_shape, dtype=torch.float32)
    if plan.empty:
        out.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
        return out, lse
    a = _cabi.WindowFwdArgs.from_buffer_copy(plan.args)
    a.q, a.k, a.v, a.out = at = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if (at[0] | at[1] | at[2] | at[3]) % 16:
        return None
    if lse is not None:
        a.lse = lse.data_ptr()
    if lens is not None:
        a.kv_lens = lens.data_ptr()
    if table is not None:
        a.page_table = table.data_ptr()
    if tree is not None:
        a.tree_mask = tree.data_ptr()
    if plan.workspace:
        workspace = q.new_empty(plan.workspace, dtype=torch.float32)
        a.joins = w = workspace.data_ptr()
        a.partial_o, a.partial_lse = w + plan.partial_o, w + plan.partial_lse
    device = q.device
    a.status = _cabi.status_buffer(device).data_ptr()
    _cabi.launch(_cabi.load().bsa_window_fwd, "bsa_window_fwd", device, a)
    return out, lse


def _check_buffers(plan: _Plan, *tensors) -> None:
    """What the caller's buffers may share memory with; ``tensors`` in the order of ``plan.apart``."""
    check_apart(plan.apart, [0 if t is None else t.data_ptr() for t in tensors])


def _copied(call, q, k, v, out, lse, layout):
    """Repeats a call on addressable copies of what the kernels cannot address; ``call(q, k, v)`` returns (out, lse)."""
    got, got_lse = call(_aligned(q, layout), k, v)
    if out is not None:
        got = out.copy_(got)
    if lse is not None:
        got_lse = lse.copy_(got_lse)
    return got, got_lse


@functools.lru_cache(maxsize=256, typed=True)
def _window_plan(q, k, v, out, lse, lens, window, sinks, softmax_scale, layout, want_lse) -> _Plan:
    window, sinks = _check_window(window, sinks)
    _check_qkv(q, k, v, layout)
    B, Hq, Hkv, Sq, Sk, D = shape = _check_shapes(q[0], k[0], v[0], layout)
    if lens is not None:
        _check_lens(lens, B, q[3], "kv_lens")
    # one head's queries do not fill a 128-row tile: tiles of several heads then, so that the group reads its keys once
    pack = Hq > Hkv and Sq < 128 and Hq // Hkv <= 128
    span = min(Sq, 128) + min(window, Sk)
    return _make_plan(q, k, v, out, lse, lens, layout, shape, window=window, sinks=sinks, scale=_check_scale(softmax_scale, D),
                      pack_gqa=pack, key_tiles=min(_ceil_div(Sk, 128), _ceil_div(span, 128) + 2), ragged=False,
                      empty=Sk == 0, want_lse=want_lse)


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

    Inside a sequence, a NaN or infinity in a value that some query sees may reach other queries of the same 128 keys;
    keys that no query sees may hold anything.  The call records no gradient: ``window_attention`` does.
    """
    want_lse = return_lse or lse is not None or q.requires_grad or k.requires_grad or v.requires_grad
    plan = _window_plan(_meta(q), _meta(k), _meta(v), _meta(out), _meta(lse), _meta(kv_lens), window, sink_tokens,
                        None if softmax_scale is None else float(softmax_scale), layout, want_lse)
    if out is not None or lse is not None:
        _check_buffers(plan, out, lse, q, k, v, kv_lens, None, None)
    res = _run_plan(plan, q, k, v, out, lse, kv_lens, None, None) if plan.direct else None
    if res is not None:
        return res
    lens = None if kv_lens is None else kv_lens.contiguous()
    return _copied(lambda q, k, v: window_attn_fwd(q, _aligned(k, layout), _aligned(v, layout), window, sink_tokens, kv_lens=lens,
                                                   softmax_scale=softmax_scale, return_lse=want_lse, layout=layout),
                   q.detach(), k.detach(), v.detach(), out, lse, layout)


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

    Gradient buffers share no memory with the inputs or with each other.  The gradients of a KV head sum over the query heads that share it, in fp32 and in a fixed order, so repeated calls
    are bit-identical.  Tokens behind ``kv_lens`` get zero gradients.  ``out`` and ``lse`` are those of the forward call
    with the same arguments.
    """
    plan = _bwd_plan(_meta(dout), _meta(q), _meta(k), _meta(v), _meta(out), _meta(lse), _meta(kv_lens), _meta(dq), _meta(dk),
                     _meta(dv), window, sink_tokens, None if softmax_scale is None else float(softmax_scale), layout)
    if dq is not None or dk is not None or dv is not None:
        check_apart(plan.apart, [0 if t is None else t.data_ptr() for t in (dq, dk, dv, dout, q, k, v, out, lse, kv_lens)])
    if not plan.direct:
        return _bwd_copied(dout, q, k, v, out, lse, window, sink_tokens, kv_lens, softmax_scale, dq, dk, dv, layout)
    grads = (q.new_empty(plan.q_shape) if dq is None else dq, q.new_empty(plan.k_shape) if dk is None else dk,
             q.new_empty(plan.k_shape) if dv is None else dv)
    if plan.empty:
        for g in grads:
            g.zero_()
        return grads
    a = _cabi.WindowBwdArgs.from_buffer_copy(plan.args)
    a.dout, a.q, a.k, a.v, a.out = at = dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.dq, a.dk, a.dv = to = grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr()
    if (at[0] | at[1] | at[2] | at[3] | at[4] | to[0] | to[1] | to[2]) % 16:
        return _bwd_copied(dout, q, k, v, out, lse, window, sink_tokens, kv_lens, softmax_scale, dq, dk, dv, layout)
    a.lse = lse.data_ptr()
    if kv_lens is not None:
        a.kv_lens = kv_lens.data_ptr()
    workspace = q.new_empty(plan.workspace, dtype=torch.uint8)
    device = q.device
    a.workspace, a.status = workspace.data_ptr(), _cabi.status_buffer(device).data_ptr()
    _cabi.launch(_cabi.load().bsa_window_bwd, "bsa_window_bwd", device, a)
    return grads


def _bwd_copied(dout, q, k, v, out, lse, window, sink_tokens, kv_lens, softmax_scale, dq, dk, dv, layout):
    """Repeats a call on addressable copies of what the kernels cannot address."""
    dout, q, k, v, out = (_aligned(t.detach(), layout) for t in (dout, q, k, v, out))
    res = window_attn_bwd(dout, q, k, v, out, lse.contiguous(), window, sink_tokens,
                          kv_lens=None if kv_lens is None else kv_lens.contiguous(), softmax_scale=softmax_scale, layout=layout)
    return tuple(g if buf is None else buf.copy_(g) for g, buf in zip(res, (dq, dk, dv)))


class _BwdPlan(NamedTuple):
    """A checked backward call: everything but the addresses."""

    direct: bool
    empty: bool
    q_shape: tuple
    k_shape: tuple
    args: bytes
    workspace: int  # bytes
    apart: tuple  # of overlap.check_apart: dq, dk, dv, dout, q, k, v, out, lse, kv_lens


@functools.lru_cache(maxsize=256, typed=True)
def _bwd_plan(dout, q, k, v, out, lse, lens, dq, dk, dv, window, sinks, softmax_scale, layout) -> _BwdPlan:
    window, sinks = _check_window(window, sinks)
    _check_qkv(q, k, v, layout)
    device = q[3]
    assert out[2] == dout[2] == q[2] and lse[2] == torch.float32, "out and dout must have q's dtype, lse float32"
    assert out[3] == dout[3] == lse[3] == device, "all tensors must be on the device of q"
    assert out[0] == q[0] and dout[0] == q[0], "out and dout must have q's shape"
    B, Hq, Hkv, Sq, Sk, D = _check_shapes(q[0], k[0], v[0], layout)
    assert lse[0] == (B, Hq, Sq), f"lse must have shape ({B}, {Hq}, {Sq})"
    if lens is not None:
        _check_lens(lens, B, device, "kv_lens")
    scale = _check_scale(softmax_scale, D)
    for buf, like in ((dq, q), (dk, k), (dv, v)):
        assert buf is None or (buf[0] == like[0] and buf[2] == like[2] and buf[3] == device and spread(*buf[:2])), (
            "gradient buffers must match q, k, v and not overlap themselves")
    q_shape, k_shape = tuple(q[0]), tuple(k[0])
    apart = pairs_apart((("dq", dq), ("dk", dk), ("dv", dv)), (("dout", dout), ("q", q), ("k", k), ("v", v), ("out", out),
                                                               ("lse", lse), ("kv_lens", lens)))
    if 0 in q_shape or 0 in k_shape:
        return _BwdPlan(True, True, q_shape, k_shape, b"", 0, apart)
    contiguous = lambda n: (n[1] * n[2] * n[3], n[2] * n[3], n[3], 1)  # noqa: E731
    grad_st = [like if buf is None else buf[1] for buf, like in ((dq, contiguous(q_shape)), (dk, contiguous(k_shape)), (dv, contiguous(k_shape)))]
    strides = [t[1] for t in (dout, q, k, v, out)] + grad_st
    if not (all(map(_fits, strides)) and _dense(lse) and (lens is None or _dense(lens))):
        return _BwdPlan(False, False, q_shape, k_shape, b"", 0, apart)
    ws = max(16, int(_cabi.load().bsa_window_bwd_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, window, sinks)))
    args = _cabi.WindowBwdArgs(*[None] * 12, ws, *(_bhsd(st, layout) for st in strides), _dtype_code(q[2]), B, Hq, Hkv, Sq, Sk, D,
                               window, sinks, scale)
    return _BwdPlan(True, False, q_shape, k_shape, bytes(args), ws, apart)


class WindowAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sink_tokens, kv_lens, softmax_scale, layout):
        out, lse = window_attn_fwd(q, k, v, window, sink_tokens, kv_lens=kv_lens, softmax_scale=softmax_scale,
                                   return_lse=True, layout=layout)
        ctx.save_for_backward(q, k, v, out, lse, kv_lens)
        ctx.how = (window, sink_tokens, softmax_scale, layout)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lens = ctx.saved_tensors
        window, sink_tokens, softmax_scale, layout = ctx.how
        dq, dk, dv = window_attn_bwd(dout, q, k, v, out, lse, window, sink_tokens, kv_lens=kv_lens,
                                     softmax_scale=softmax_scale, layout=layout)
        return dq, dk, dv, None, None, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sink_tokens: int = 0,
                     kv_lens: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                     layout: str = "bhsd") -> torch.Tensor:
    """Differentiable sliding-window attention with sinks (see ``window_attn_fwd`` for the arguments).

    Once differentiable.  To capture a training step in a CUDA graph, warm it up on a side stream and drop every eager
    graph of the same leaves first, as PyTorch asks for any captured backward pass."""
    return WindowAttentionFunction.apply(q, k, v, window, sink_tokens, kv_lens, softmax_scale, layout)
