"""Rotary positions with several axes (text; height and width of images; time, height and width of videos).

Applied to q and k before any of the framework's attention operators (the reference has no counterpart).  The rotation's
backward pass is the rotation by the opposite angles, so ``rotary_nd(..., inverse=True)`` is it.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _cabi
from .overlap import check_apart, pairs_apart, spread
from .window_attn import _meta

__all__ = ["rotary_frequencies", "rotary_nd", "rotary_embedding", "RotaryFunction"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 2, torch.float32: 3}


def rotary_frequencies(axis_pairs: Sequence[int], theta: float = 10000.0, *, shared_ladder: bool = False,
                       device: Optional[torch.device] = None) -> torch.Tensor:
    """fp32 ``inv_freq[sum(axis_pairs)]``: pair ``i`` of an axis with ``n`` pairs turns at ``theta ** (-i / n)``; with
    ``shared_ladder`` one ladder over all pairs is dealt to the axes in order."""
    assert len(axis_pairs) >= 1 and all(int(n) >= 0 for n in axis_pairs) and theta > 0
    counts = [sum(axis_pairs)] if shared_ladder else list(axis_pairs)
    parts = [float(theta) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in counts]
    return torch.cat(parts).to(device=device, dtype=torch.float32)


def rotary_nd(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    axis_pairs: Sequence[int],
    *,
    interleaved: bool = True,
    inverse: bool = False,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
    layout: str = "bhsd",
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotates q and (unless None) k; returns ``(q_rotated, k_rotated_or_None)``.

    ``q`` is ``[B, Hq, S, D]``, ``k`` ``[B, Hk, S, D]`` (``layout="bshd"``: heads and tokens swapped), BF16, FP16 or FP32, ``D``
    even and at most 512; any strides whose last is 1.  The first ``2 * P`` channels of a head turn, ``P =
    sum(axis_pairs)``, the others are copied.  Pair ``p`` is channels ``(2p, 2p + 1)``, or ``(p, P + p)`` with
    ``interleaved=False``; it belongs to the axis whose share of ``axis_pairs`` (1 to 4 axes, in order) holds ``p`` and turns
    by ``positions[b, s, axis] * inv_freq[p]`` (``inverse=True``: by the opposite angle).  ``positions`` is int32
    ``[S, axes]`` or ``[B, S, axes]``, ``inv_freq`` fp32 ``[P]`` (``rotary_frequencies``).  Angles are reduced in 64 bits, so
    positions of any size keep their accuracy.  ``q_out`` / ``k_out`` may be q and k themselves (in place); outputs that share
    other memory are refused.  The call records no gradient: ``rotary_embedding`` does.
    """
    pairs = tuple(map(int, axis_pairs))
    plan = _rotary_plan(_meta(q), _meta(k), _meta(positions), _meta(inv_freq), pairs, bool(interleaved), bool(inverse),
                        _meta(q_out), _meta(k_out), layout)
    if q_out is not None or k_out is not None:
        check_apart(plan.apart, [0 if t is None else t.data_ptr() for t in (q_out, k_out, q, k, positions, inv_freq)])
    if not plan.direct:
        return rotary_nd(q if q.stride(3) == 1 else q.contiguous(), k if k is None or k.stride(3) == 1 else k.contiguous(),
                         positions.contiguous(), inv_freq.contiguous(), pairs, interleaved=interleaved, inverse=inverse,
                         q_out=q_out, k_out=k_out, layout=layout)
    if q_out is None:
        q_out = torch.empty_like(q) if plan.q_dense else q.new_empty(plan.q_shape)
    if k is None:
        k_out = None
    elif k_out is None:
        k_out = torch.empty_like(k) if plan.k_dense else q.new_empty(plan.k_shape)
    if plan.empty:
        return q_out, k_out
    a = _cabi.RotaryArgs.from_buffer_copy(plan.args)
    a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
    if k is not None:
        a.k, a.k_out = k.data_ptr(), k_out.data_ptr()
    a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    _cabi.launch(_cabi.load().bsa_rotary_nd, "bsa_rotary_nd", q.device, a)
    return q_out, k_out


def _contiguous(t) -> bool:
    n = t[0]
    return t[1] == (n[1] * n[2] * n[3], n[2] * n[3], n[3], 1)


class _RotaryPlan(NamedTuple):
    """A checked call: everything but the addresses, kept as in ``window_attn._Plan``."""

    direct: bool  # unit last strides
    empty: bool
    q_shape: tuple
    k_shape: Optional[tuple]
    args: bytes
    apart: tuple  # of overlap.check_apart: q_out, k_out, q, k, positions, inv_freq
    q_dense: bool = False  # contiguous: empty_like, the cheaper call, gives the same
    k_dense: bool = False


@functools.lru_cache(maxsize=256, typed=True)
def _rotary_plan(q, k, positions, inv_freq, pairs, interleaved, inverse, q_out, k_out, layout) -> _RotaryPlan:
    assert layout in ("bhsd", "bshd"), f"layout must be 'bhsd' or 'bshd', got {layout!r}"
    assert len(q[0]) == 4 and q[4], "q must be a 4-D CUDA tensor"
    code, device = _DTYPES.get(q[2]), q[3]
    assert code is not None, "q must be bfloat16, float16 or float32"
    h, s = (1, 2) if layout == "bhsd" else (2, 1)  # dimensions of heads and tokens
    B, Hq, S, D = q[0][0], q[0][h], q[0][s], q[0][3]
    assert D % 2 == 0 and 2 <= D <= 512, f"head dimension must be even and at most 512, got {D}"
    P, A = sum(pairs), len(pairs)
    assert 1 <= A <= 4 and min(pairs) >= 0 and 1 <= P and 2 * P <= D, (
        f"axis_pairs {pairs} must be 1 to 4 axes with 1 to {D // 2} pairs in all")
    Hk = 0
    if k is not None:
        assert len(k[0]) == 4 and k[2] == q[2] and k[3] == device, "k must match q's type and device"
        Hk = k[0][h]
        assert k[0][0] == B and k[0][s] == S and k[0][3] == D, "k must match q's batch, tokens and head dimension"
    assert positions[2] == torch.int32 and positions[3] == device, "positions must be int32 on the device of q"
    at = tuple(positions[0])
    assert at == (S, A) or at == (B, S, A), f"positions has shape {at}, expected ({S}, {A}) or ({B}, {S}, {A})"
    assert inv_freq[2] == torch.float32 and inv_freq[3] == device and inv_freq[0] == (P,), (
        f"inv_freq must be float32 of shape ({P},) on the device of q")
    for name, x, out in (("q_out", q, q_out), ("k_out", k, k_out)):
        if out is not None:
            assert x is not None and out[0] == x[0] and out[2] == x[2] and out[3] == device, f"{name} must match its input"
            assert out[1][3] == 1 and spread(*out[:2]), f"{name} must have unit last stride and not overlap itself"
    q_shape, k_shape = tuple(q[0]), None if k is None else tuple(k[0])
    apart = pairs_apart((("q_out", q_out), ("k_out", k_out)), (("q", q), ("k", k), ("positions", positions), ("inv_freq", inv_freq)),
                        (("q_out", "q"), ("k_out", "k")))
    if B == 0 or S == 0 or (Hq == 0 and Hk == 0):
        return _RotaryPlan(True, True, q_shape, k_shape, b"", apart)
    assert Hq >= 1, "q has no heads"
    if q[1][3] != 1 or (Hk > 0 and k[1][3] != 1) or (A > 1 and positions[1][-1] != 1) or (P > 1 and inv_freq[1] != (1,)):
        return _RotaryPlan(False, False, q_shape, k_shape, b"", apart)

    def strides(t, out=None):
        if t is None:
            return 0, 0, 0
        if out is None:  # a fresh contiguous tensor of t's shape
            n = t[0]
            st = (n[1] * n[2] * n[3], n[2] * n[3], n[3])
        else:
            st = out[1]
        return st[0], st[h], st[s]

    pos_st = positions[1]
    args = _cabi.RotaryArgs(None, None, None, None, None, None, strides(q, q), strides(k, k), strides(q, q_out), strides(k, k_out),
                            (pos_st[0] if len(at) == 3 else 0, pos_st[-2]), pairs, A, code, B, Hq, Hk, S, D, int(interleaved),
                            int(inverse))
    return _RotaryPlan(True, False, q_shape, k_shape, bytes(args), apart, _contiguous(q), k is not None and _contiguous(k))


class RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axis_pairs, interleaved, layout):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (tuple(axis_pairs), interleaved, layout)
        ctx.set_materialize_grads(False)
        return rotary_nd(q, k, positions, inv_freq, axis_pairs, interleaved=interleaved, layout=layout)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        pairs, interleaved, layout = ctx.how
        how = dict(interleaved=interleaved, layout=layout, inverse=True)
        if dq is None and dk is not None:
            dk = rotary_nd(dk, None, positions, inv_freq, pairs, **how)[0]
        elif dq is not None:
            dq, dk = rotary_nd(dq, dk, positions, inv_freq, pairs, **how)
        return dq, dk, None, None, None, None, None


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
                     axis_pairs: Sequence[int], interleaved: bool = True, layout: str = "bhsd"
                     ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Differentiable ``rotary_nd`` (with respect to q and k).  Once differentiable; captured in a CUDA graph as
    ``window_attention`` is."""
    return RotaryFunction.apply(q, k, positions, inv_freq, axis_pairs, interleaved, layout)
