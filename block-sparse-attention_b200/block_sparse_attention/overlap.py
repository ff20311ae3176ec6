"""Whether strided views share memory: a call refuses outputs that meet one of its inputs or another output.

The spans of two views decide nearly every case.  Views whose spans interleave (slices of one fused projection, key and
value pages of one pool) are compared exactly.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Sequence, Tuple

__all__ = ["span_bytes", "spread", "same_places", "pairs_apart", "check_apart"]

_MOST_STEPS = 20000  # of the exact comparison; views that need more (strides that do not nest) count as meeting


def span_bytes(shape, strides, size: int) -> int:
    """Bytes from a view's first element to behind its last; 0 for an empty one."""
    return 0 if 0 in shape else (sum((n - 1) * s for n, s in zip(shape, strides)) + 1) * size


def spread(shape, strides) -> bool:
    """Whether every element has a place of its own (strides that nest, as those of slices and transposes do)."""
    end = 1
    for s, n in sorted((s, n) for s, n in zip(strides, shape) if n > 1):
        if s < end:
            return 0 in shape
        end += s * (n - 1)
    return True


def same_places(a, b) -> bool:
    """Whether two (shape, strides) put every element at the same place; a dimension of size 1 may have any stride."""
    return a[0] == b[0] and all(n == 1 or s == t for n, s, t in zip(a[0], a[1], b[1]))


def _runs(shape, strides, size: int) -> Tuple[int, list]:
    """A view as runs of bytes: their length, and (stride, number) of what repeats them."""
    run, dims = size, []
    for s, n in sorted((s * size, n) for s, n in zip(strides, shape) if n > 1 and s > 0):
        if not dims and s <= run:
            run += s * (n - 1)
        else:
            dims.append((s, n))
    return run, dims


@functools.lru_cache(maxsize=256)
def _meet(a, b, distance: int) -> bool:
    """``a``, ``b`` are (shape, strides, element size), b's first element lies ``distance`` bytes behind a's."""
    (a_run, a_dims), (b_run, b_dims) = _runs(*a), _runs(*b)
    # some byte is in both iff sum i s - sum j t lies between distance - a_run and distance + b_run for some indices i of a's
    # repeats (strides s) and j of b's (strides t); one multiple for each stride
    least, most = {}, {}
    for s, n in a_dims:
        least[s], most[s] = least.get(s, 0), most.get(s, 0) + n - 1
    for s, n in b_dims:
        least[s], most[s] = least.get(s, 0) - (n - 1), most.get(s, 0)
    terms = sorted(least, reverse=True)
    below, above = [0], [0]  # range of the sums of the last terms
    for s in reversed(terms):
        below.append(below[-1] + s * least[s])
        above.append(above[-1] + s * most[s])
    below.reverse()
    above.reverse()
    steps = 0

    def solve(k: int, lo: int, hi: int) -> bool:
        nonlocal steps
        steps += 1
        if k == len(terms):
            return lo < 0 < hi
        if steps > _MOST_STEPS:
            return True
        s = terms[k]
        first = max(least[s], (lo - above[k + 1]) // s + 1)
        last = min(most[s], -((below[k + 1] - hi) // s) - 1)
        return any(solve(k + 1, lo - s * m, hi - s * m) for m in range(first, last + 1))

    return solve(0, distance - a_run, distance + b_run)


class _Pair(NamedTuple):
    out: int  # places in the list of addresses
    other: int
    out_span: int
    other_span: int
    views: tuple
    may_be_one: bool
    names: str


def pairs_apart(outputs: Sequence[Tuple[str, Optional[tuple]]], inputs: Sequence[Tuple[str, Optional[tuple]]],
                in_place: Sequence[Tuple[str, str]] = ()) -> Tuple[_Pair, ...]:
    """What ``check_apart`` looks at, from the tensors' (shape, strides, dtype, ...), None where there is none: each output beside
    the outputs behind it and every input.  The pairs ``in_place`` (output, input) may be one and the same view."""
    views = [None if m is None else (tuple(m[0]), tuple(m[1]), m[2].itemsize) for _, m in (*outputs, *inputs)]
    names = [name for name, _ in (*outputs, *inputs)]
    spans = [0 if v is None else span_bytes(*v) for v in views]
    return tuple(_Pair(i, j, spans[i], spans[j], (views[i], views[j]),
                       (names[i], names[j]) in in_place and views[i][2] == views[j][2] and same_places(views[i], views[j]),
                       f"{names[i]} and {names[j]} must not share memory")
                 for i in range(len(outputs)) for j in range(i + 1, len(views)) if spans[i] and spans[j])


def check_apart(pairs: Tuple[_Pair, ...], addresses: Sequence[int]) -> None:
    """Refuses outputs that share memory with another output or an input; addresses in the order of ``pairs_apart``'s arguments
    (anything for a tensor that there is not)."""
    for i, j, out_span, other_span, views, may_be_one, names in pairs:
        distance = addresses[j] - addresses[i]
        if -other_span < distance < out_span:
            assert (may_be_one and distance == 0) or not _meet(*views, distance), names
