"""Rotary positions with several axes (text; height and width of images; time, height and width of videos).

Applied to q and k before any of the framework's attention operators (the reference has no counterpart).  The rotation's
backward pass is the rotation by the opposite angles, so ``rotary_nd(..., inverse=True)`` is it.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _cabi

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


def _span(t: torch.Tensor) -> Tuple[int, int]:
    end = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (end + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


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
    positions of any size keep their accuracy.  ``q_out`` / ``k_out`` may be q and k themselves (in place); other overlaps
    are refused.
    """
    assert layout in ("bhsd", "bshd"), f"layout must be 'bhsd' or 'bshd', got {layout!r}"
    assert q.dim() == 4 and q.is_cuda, "q must be a 4-D CUDA tensor"
    code = _DTYPES.get(q.dtype)
    assert code is not None, "q must be bfloat16, float16 or float32"
    device = q.device
    h, s = (1, 2) if layout == "bhsd" else (2, 1)  # dimensions of heads and tokens
    shape = q.shape
    B, Hq, S, D = shape[0], shape[h], shape[s], shape[3]
    assert D % 2 == 0 and 2 <= D <= 512, f"head dimension must be even and at most 512, got {D}"
    pairs = tuple(axis_pairs)
    P, A = sum(pairs), len(pairs)
    assert 1 <= A <= 4 and min(pairs) >= 0 and 1 <= P and 2 * P <= D, (
        f"axis_pairs {pairs} must be 1 to 4 axes with 1 to {D // 2} pairs in all")
    Hk = 0
    if k is not None:
        assert k.dim() == 4 and k.dtype == q.dtype and k.device == device, "k must match q's type and device"
        Hk = k.shape[h]
        assert k.shape[0] == B and k.shape[s] == S and k.shape[3] == D, "k must match q's batch, tokens and head dimension"
    assert positions.dtype == torch.int32 and positions.device == device, "positions must be int32 on the device of q"
    at = tuple(positions.shape)
    assert at == (S, A) or at == (B, S, A), f"positions has shape {at}, expected ({S}, {A}) or ({B}, {S}, {A})"
    assert inv_freq.dtype == torch.float32 and inv_freq.device == device and tuple(inv_freq.shape) == (P,), (
        f"inv_freq must be float32 of shape ({P},) on the device of q")
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    inv_freq = inv_freq.contiguous()
    qo, ko = q_out, k_out
    if q.stride(3) != 1:
        q = q.contiguous()
    if k is not None and k.stride(3) != 1:
        k = k.contiguous()
    if q_out is None:
        qo = torch.empty_like(q)
    if k is None:
        ko = None
    elif k_out is None:
        ko = torch.empty_like(k)
    if q_out is not None or (k is not None and k_out is not None):  # fresh outputs overlap nothing
        _check_outputs(q, qo, k, ko)
    if B == 0 or S == 0 or (Hq == 0 and Hk == 0):
        return qo, ko
    assert Hq >= 1, "q has no heads"
    zero = (0, 0, 0)

    def strides(t):
        if t is None:
            return zero
        st = t.stride()
        return st[0], st[h], st[s]

    pos_st = positions.stride()
    a = _cabi.RotaryArgs(
        q.data_ptr(), None if k is None else k.data_ptr(), qo.data_ptr(), None if k is None else ko.data_ptr(),
        positions.data_ptr(), inv_freq.data_ptr(), strides(q), strides(k), strides(qo), strides(ko),
        (pos_st[0] if len(at) == 3 else 0, pos_st[-2]), pairs, A, code, B, Hq, Hk, S, D, 1 if interleaved else 0,
        1 if inverse else 0)
    _cabi.launch(_cabi.load().bsa_rotary_nd, "bsa_rotary_nd", device, a)
    return qo, ko


def _check_outputs(q, qo, k, ko) -> None:
    for name, x, out in (("q_out", q, qo), ("k_out", k, ko)):
        if out is not None:
            assert out.shape == x.shape and out.dtype == x.dtype and out.device == x.device, f"{name} must match its input"
            assert out.stride(-1) == 1 and all(n == 1 or st > 0 for n, st in zip(out.shape, out.stride())), (
                f"{name} must have unit last stride and no broadcast dimension")
    if any(t is not None and t.numel() == 0 for t in (q, k)):
        return
    for out, own, other, other_out in ((qo, q, k, ko), (ko, k, q, qo)):
        if out is None:
            continue
        assert _same_view(out, own) or not _overlap(out, own), "an output may be its input or apart from it, not overlap it"
        if other is not None:
            # views of one fused projection may interleave; then both have to be rotated in place
            apart = not _overlap(out, other) and not _overlap(out, other_out)
            assert apart or (_same_view(out, own) and _same_view(other_out, other) and out.data_ptr() != other.data_ptr()), (
                "q and k and their outputs must not overlap, unless both are rotated in place")


class RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axis_pairs, interleaved, layout):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (tuple(axis_pairs), interleaved, layout)
        ctx.set_materialize_grads(False)
        return rotary_nd(q, k, positions, inv_freq, axis_pairs, interleaved=interleaved, layout=layout)

    @staticmethod
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
    """Differentiable ``rotary_nd`` (with respect to q and k)."""
    return RotaryFunction.apply(q, k, positions, inv_freq, axis_pairs, interleaved, layout)
