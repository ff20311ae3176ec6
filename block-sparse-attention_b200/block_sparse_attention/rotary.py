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
    assert q.dtype in _DTYPES, "q must be bfloat16, float16 or float32"
    assert k is None or (k.dim() == 4 and k.dtype == q.dtype and k.device == q.device), "k must match q's type and device"
    device = q.device
    tr = (lambda t: t) if layout == "bhsd" else (lambda t: t.transpose(1, 2))
    pairs = [int(n) for n in axis_pairs]
    P = sum(pairs)
    B, Hq, S, D = tr(q).shape
    assert D % 2 == 0 and 2 <= D <= 512, f"head dimension must be even and at most 512, got {D}"
    assert 1 <= len(pairs) <= 4 and min(pairs) >= 0 and 1 <= P and 2 * P <= D, (
        f"axis_pairs {tuple(pairs)} must be 1 to 4 axes with 1 to {D // 2} pairs in all")
    if k is not None:
        assert tr(k).shape[0] == B and tr(k).shape[2:] == (S, D), "k must match q's batch, tokens and head dimension"
    assert positions.dtype == torch.int32 and positions.device == device, "positions must be int32 on the device of q"
    assert tuple(positions.shape) in ((S, len(pairs)), (B, S, len(pairs))), (
        f"positions has shape {tuple(positions.shape)}, expected ({S}, {len(pairs)}) or ({B}, {S}, {len(pairs)})")
    assert inv_freq.dtype == torch.float32 and inv_freq.device == device and tuple(inv_freq.shape) == (P,), (
        f"inv_freq must be float32 of shape ({P},) on the device of q")
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    inv_freq = inv_freq.contiguous()

    def prepare(x, out, name):
        x = x if x.stride(-1) == 1 else x.contiguous()
        if out is None:
            return x, torch.empty(x.shape, dtype=x.dtype, device=device)
        assert out.shape == x.shape and out.dtype == x.dtype and out.device == device, f"{name} must match its input"
        assert out.stride(-1) == 1 and all(n == 1 or s > 0 for n, s in zip(out.shape, out.stride())), (
            f"{name} must have unit last stride and no broadcast dimension")
        return x, out

    q, qo = prepare(q, q_out, "q_out")
    k, ko = (None, None) if k is None else prepare(k, k_out, "k_out")
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return qo, ko
    for out, own, other, other_out in ((qo, q, k, ko), (ko, k, q, qo)):
        if out is None:
            continue
        assert _same_view(out, own) or not _overlap(out, own), "an output may be its input or apart from it, not overlap it"
        if other is not None:
            # views of one fused projection may interleave; then both have to be rotated in place
            apart = not _overlap(out, other) and not _overlap(out, other_out)
            assert apart or (_same_view(out, own) and _same_view(other_out, other) and out.data_ptr() != other.data_ptr()), (
                "q and k and their outputs must not overlap, unless both are rotated in place")
    a = _cabi.RotaryArgs()
    qv, qov = tr(q), tr(qo)
    a.q, a.q_out = qv.data_ptr(), qov.data_ptr()
    a.q_stride, a.qo_stride = _cabi.strides3(qv), _cabi.strides3(qov)
    if k is not None:
        kv, kov = tr(k), tr(ko)
        a.k, a.k_out = kv.data_ptr(), kov.data_ptr()
        a.k_stride, a.ko_stride = _cabi.strides3(kv), _cabi.strides3(kov)
        a.Hk = kv.shape[1]
    a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    a.pos_stride[0] = positions.stride(0) if positions.dim() == 3 else 0
    a.pos_stride[1] = positions.stride(-2)
    for i, n in enumerate(pairs):
        a.axis_pairs[i] = n
    a.num_axes = len(pairs)
    a.dtype = _DTYPES[q.dtype]
    a.B, a.Hq, a.S, a.D = B, Hq, S, D
    a.interleaved, a.inverse = int(bool(interleaved)), int(bool(inverse))
    with torch.cuda.device(device):
        _cabi.check(_cabi.load().bsa_rotary_nd(a, _cabi.stream_ptr(device)), "bsa_rotary_nd")
    return qo, ko


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
