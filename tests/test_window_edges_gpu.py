"""GPU parity of sliding-window attention at its edges: what rows hold that take no part, first rows, unbounded lengths, buffers."""
import pytest
import torch

from dealing import DEALS, deal  # noqa: F401
from plain_ops import assert_close_norm, assert_within, attend, gradients, half_step
from test_window_gpu import BF, HF, make, masks

pytestmark = pytest.mark.gpu


def i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


# B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, lens
CHUNKS = [
    (1, 2, 2, 100, 500, 128, BF, 50, 3, None),       # keys between the sinks and the first window
    (2, 6, 2, 130, 700, 64, HF, 200, 0, [700, 640]),
    (1, 2, 1, 300, 1000, 96, BF, 300, 70, None),     # more sinks than the narrow tile's columns
    (1, 4, 1, 1, 400, 128, HF, 128, 128, None),      # one query, sinks up to the tile's end
    (2, 2, 2, 40, 129, 64, BF, 1, 0, [129, 100]),
    (1, 40, 40, 200, 900, 64, BF, 260, 33, None),
]


def poison_unseen(k, v, mask, holds):
    """k, v [B, H, S, D] with `holds` in the keys that no row of mask [B, Sq, S] sees."""
    unseen = ~mask.any(1)[:, None, :, None]
    assert unseen.any()
    return k.masked_fill(unseen, holds), v.masked_fill(unseen, holds)


@pytest.mark.parametrize("deal", DEALS, indirect=True, ids=str)
@pytest.mark.parametrize("case", CHUNKS, ids=[str(i) for i in range(len(CHUNKS))])
def test_keys_before_every_window_may_hold_anything(case, deal):
    from block_sparse_attention import window_attn_fwd
    B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, lens = case
    q, k, v, _ = make(B, Hq, Hkv, Sq, Sk, D, dtype, seed=3)
    mask = masks(B, Sq, Sk, window, sinks, lens)
    ref, lse, tol, lse_tol, _, _ = attend(q.double(), k.double(), v.double(), mask, D ** -0.5, dtype)
    for holds in (float("nan"), float("inf")):
        kp, vp = poison_unseen(k, v, mask, holds)
        out, got = window_attn_fwd(q.cuda(), kp.cuda(), vp.cuda(), window, sinks, kv_lens=i32(lens), return_lse=True)
        assert_within(out, ref, tol, "out")
        assert_within(got, lse, lse_tol, "lse")


@pytest.mark.parametrize("case", CHUNKS, ids=[str(i) for i in range(len(CHUNKS))])
def test_gradients_with_anything_in_keys_before_every_window(case):
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, lens = case
    q, k, v, do = make(B, Hq, Hkv, Sq, Sk, D, dtype, seed=4)
    mask = masks(B, Sq, Sk, window, sinks, lens)
    refs, tols = gradients(q.double(), k.double(), v.double(), do.double(), mask, D ** -0.5, dtype)
    n = i32(lens)
    for holds in (float("nan"), float("inf")):
        kp, vp = (t.cuda() for t in poison_unseen(k, v, mask, holds))
        out, lse = window_attn_fwd(q.cuda(), kp, vp, window, sinks, kv_lens=n, return_lse=True)
        grads = window_attn_bwd(do.cuda(), q.cuda(), kp, vp, out, lse, window, sinks, kv_lens=n)
        for name, g, ref, tol in zip(("dq", "dk", "dv"), grads, refs, tols):
            assert_within(g, ref, tol, name)


# more queries than keys: the first ones sit before the first key
LATE = [
    (1, 2, 2, 200, 100, 64, BF, 40, 2),
    (2, 6, 2, 400, 150, 128, HF, 1 << 20, 0),
    (1, 40, 40, 700, 260, 96, BF, 100, 5),   # many key tiles: not cut into parts
    (3, 2, 1, 30, 7, 64, HF, 3, 0),          # a few visible keys
]


@pytest.mark.parametrize("case", LATE, ids=[str(i) for i in range(len(LATE))])
def test_queries_before_the_first_key_may_hold_anything(case):
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks = case
    q, k, v, do = make(B, Hq, Hkv, Sq, Sk, D, dtype, seed=5)
    mask = masks(B, Sq, Sk, window, sinks, None)
    refs, tols = gradients(q.double(), k.double(), v.double(), do.double(), mask, D ** -0.5, dtype)
    ref, rl, tol, lt, _, _ = attend(q.double(), k.double(), v.double(), mask, D ** -0.5, dtype)
    for holds in (float("nan"), float("inf")):
        for t in (q, do):
            t[:, :, :Sq - Sk] = holds
        out, lse = window_attn_fwd(q.cuda(), k.cuda(), v.cuda(), window, sinks, return_lse=True)
        assert_within(out, ref, tol, "out")
        assert_within(lse, rl, lt, "lse")
        grads = window_attn_bwd(do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, window, sinks)
        for name, g, want, t in zip(("dq", "dk", "dv"), grads, refs, tols):
            assert_within(g, want, t, name)


@pytest.mark.parametrize("Sq,Sk", [(200, 100), (150, 150), (40, 300), (60, 9)])
def test_a_length_without_a_limit_is_the_whole_sequence(Sq, Sk):
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    q, k, v, do = (t.cuda() for t in make(2, 4, 2, Sq, Sk, 64, BF, seed=6))

    def step(n):
        out, lse = window_attn_fwd(q, k, v, 40, 2, kv_lens=n, return_lse=True)
        return (out, lse) + window_attn_bwd(do, q, k, v, out, lse, 40, 2, kv_lens=n)

    want = step(None)
    assert all(t.any() for t in want)
    for n in (2 ** 31 - 1, 2 ** 31 - 40, Sk + 1, Sk):
        assert all(torch.equal(a, b) for a, b in zip(step(i32([n, n])), want)), n


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Sq,Sk,window,sinks,lens", [
    (64, 64, 100, 3, None), (65, 65, 100, 3, None), (1000, 1000, 100, 3, None),  # wherever the sequence ends
    (300, 302, 4, 2, None), (299, 303, 6, 0, None), (200, 90, 3, 100, None),     # the first rows at 2, 4 and -110
    (128, 128, 70, 0, 4), (4, 4, 70, 0, None), (128, 128, 2, 4, 3),              # short sequences, padded and not
])
def test_first_rows_keep_their_gradients(Sq, Sk, window, sinks, lens, dtype):
    """delta nearly cancels dP in rows that see a few keys.  dS and dQ are each off by at most u / sqrt(3) in the mean
    square, u half a step: together 0.82 u."""
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    B, D = 60, 64
    q, k, v, do = make(B, 6, 2, Sq, Sk, D, dtype, seed=7)
    n = None if lens is None else [lens] * B
    first = max(0, Sq - Sk)
    rows = slice(first, min(Sq, first + 5 - max(0, Sk - Sq)))  # at positions below 5
    keys = slice(0, 5)
    mask = masks(B, Sq, Sk, window, sinks, n)[:, rows, keys]
    (ref, _, _), _ = gradients(q[:, :, rows].double(), k[:, :, keys].double(), v[:, :, keys].double(), do[:, :, rows].double(), mask, D ** -0.5, dtype)
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    out, lse = window_attn_fwd(q, k, v, window, sinks, kv_lens=i32(n), return_lse=True)
    dq, _, _ = window_attn_bwd(do, q, k, v, out, lse, window, sinks, kv_lens=i32(n))
    assert_close_norm(dq[:, :, rows], ref, 0.82 * half_step(dtype), "dq")


@pytest.mark.parametrize("deal", DEALS, indirect=True, ids=str)
def test_results_do_not_depend_on_what_padding_holds(deal):
    """To the bit: forward and backward, padded query rows beside live ones of the same warp."""
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    q, k, v, do = (t.cuda() for t in make(3, 4, 2, 400, 400, 128, BF, seed=8))
    lens = [200, 307, 5]
    n, got = i32(lens), []
    for holds in (0.0, 30.0, -1000.0, float("nan")):
        q2, k2, v2, do2 = q.clone(), k.clone(), v.clone(), do.clone()
        for b, m in enumerate(lens):
            for t in (q2, k2, v2, do2):
                t[b, :, m:] = t[b, :, m:] * holds
        out, lse = window_attn_fwd(q2, k2, v2, 4096, 0, kv_lens=n, return_lse=True)
        got.append((out, lse) + window_attn_bwd(do2, q2, k2, v2, out, lse, 4096, 0, kv_lens=n))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_buffers_that_interleave_without_meeting():
    """Slices of fused tensors as outputs, `out` in the place of q."""
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    B, S, H, Hkv, D = 2, 300, 4, 2, 64
    q, k, v, do = (t.transpose(1, 2).contiguous().cuda() for t in make(B, H, Hkv, S, S, D, BF, seed=9))
    how = dict(layout="bshd")
    want, lse = window_attn_fwd(q, k, v, 70, 2, return_lse=True, **how)
    fused = torch.cat((q, k, v), 2)
    parts = fused.split((H, Hkv, Hkv), 2)
    grads = window_attn_bwd(do, q, k, v, want, lse, 70, 2, **how)
    into = torch.full_like(fused, 7.0)
    slices = into.split((H, Hkv, Hkv), 2)
    window_attn_bwd(do, *parts, want, lse, 70, 2, dq=slices[0], dk=slices[1], dv=slices[2], **how)
    assert torch.equal(into, torch.cat(grads, 2))
    for sizes in ((300, 300), (300, 20)):  # whole query tiles; packed heads and shared lists
        q2 = fused[:, :sizes[1], :H]
        ref, _ = window_attn_fwd(q2.clone(), parts[1], parts[2], 70, 2, **how)
        out, _ = window_attn_fwd(q2, parts[1], parts[2], 70, 2, out=q2, **how)
        assert out is q2 and torch.equal(q2, ref) and torch.equal(parts[1], k) and torch.equal(parts[2], v)
