"""GPU parity of sliding-window attention with sinks (forward, backward) against a plain 64-bit implementation."""
import math

import pytest
import torch

from plain_ops import assert_close_norm, assert_within, attend, gradients, half_step, visible

pytestmark = pytest.mark.gpu


def make(B, Hq, Hkv, Sq, Sk, D, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q, do = ((torch.randn(B, Hq, Sq, D, generator=g) * spread).to(dtype) for _ in range(2))
    k, v = ((torch.randn(B, Hkv, Sk, D, generator=g) * spread).to(dtype) for _ in range(2))
    return q, k, v, do


def masks(B, Sq, Sk, window, sinks, lens):
    return torch.stack([visible(Sq, Sk, window, sinks, Sk if lens is None else lens[b]) for b in range(B)])


def poison(t, lens, offset):
    """Fills the tokens at positions >= lens[b] of [B, H, S, D] with NaN (token i is at i + offset)."""
    t = t.clone()
    for b, n in enumerate(lens):
        t[b, :, max(0, n - offset):] = float("nan")
    return t


BF, HF = torch.bfloat16, torch.float16
# B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, lens
CASES = [
    (1, 1, 1, 1, 1, 128, BF, 1, 0, None),
    (1, 2, 1, 1, 200, 64, HF, 64, 3, None),
    (2, 2, 2, 127, 127, 128, BF, 1, 0, None),          # every row sees itself only
    (1, 2, 2, 128, 128, 96, BF, 128, 128, None),
    (1, 4, 2, 129, 129, 128, HF, 100, 1, None),
    (1, 2, 2, 640, 640, 128, BF, 256, 4, None),         # window of whole tiles
    (1, 3, 1, 700, 700, 64, BF, 130, 100, None),        # three heads a KV head
    (2, 4, 4, 513, 513, 96, HF, 77, 0, [513, 200]),     # padded batch
    (3, 2, 1, 300, 300, 128, BF, 150, 5, [0, 1, 299]),  # sequences of no and of one token
    (1, 6, 2, 50, 900, 128, BF, 300, 4, None),          # a chunk behind a long past, packed heads, split keys
    (2, 5, 1, 33, 1000, 64, HF, 1 << 20, 0, [1000, 980]),   # five heads a KV head, window longer than all
    (1, 1, 1, 200, 100, 128, BF, 40, 2, None),          # queries before the first key
    (1, 2, 2, 1300, 1300, 128, BF, 1, 128, None),       # sinks only, and the row itself
    (1, 4, 1, 1100, 1100, 64, HF, 200, 2, None),
    (1, 1, 1, 2000, 2000, 128, BF, 1000, 4, None),      # few long lists: cut into runs in every kernel
    (2, 2, 1, 1500, 1500, 96, HF, 1 << 20, 0, [1500, 700]),
    (1, 8, 1, 6, 38, 96, BF, 24, 1, None),              # one key tile, eight heads
    (3, 2, 2, 1000, 1200, 64, BF, 900, 65, [1200, 0, 333]),
    (2, 40, 40, 1200, 1200, 64, BF, 130, 70, None),     # many items: whole ones, the sinks' beyond them
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_forward(case, layout):
    from block_sparse_attention import window_attn_fwd
    B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, lens = case
    q, k, v, _ = make(B, Hq, Hkv, Sq, Sk, D, dtype)
    ref, lse, tol, lse_tol, _, _ = attend(q.double(), k.double(), v.double(), masks(B, Sq, Sk, window, sinks, lens), D ** -0.5, dtype)
    if lens is not None:
        k, v, q = poison(k, lens, 0), poison(v, lens, 0), poison(q, lens, Sk - Sq)
    qc, kc, vc = (t.cuda() if layout == "bhsd" else t.transpose(1, 2).contiguous().cuda() for t in (q, k, v))
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    out, got_lse = window_attn_fwd(qc, kc, vc, window, sinks, kv_lens=n, return_lse=True, layout=layout)
    out = out if layout == "bhsd" else out.transpose(1, 2)
    assert_within(out, ref, tol, "out")
    assert_within(got_lse, lse, lse_tol, "lse")
    out2, none = window_attn_fwd(qc, kc, vc, window, sinks, kv_lens=n, layout=layout)
    assert none is None and torch.equal(out2 if layout == "bhsd" else out2.transpose(1, 2), out)


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_backward(case):
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    B, Hq, Hkv, Sq, Sk, D, dtype, window, sinks, lens = case
    q, k, v, do = make(B, Hq, Hkv, Sq, Sk, D, dtype, seed=1)
    mask = masks(B, Sq, Sk, window, sinks, lens)
    refs, tols = gradients(q.double(), k.double(), v.double(), do.double(), mask, D ** -0.5, dtype)
    if lens is not None:
        k, v, q, do = poison(k, lens, 0), poison(v, lens, 0), poison(q, lens, Sk - Sq), poison(do, lens, Sk - Sq)
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = window_attn_fwd(q, k, v, window, sinks, kv_lens=n, return_lse=True)
    grads = window_attn_bwd(do, q, k, v, out, lse, window, sinks, kv_lens=n)
    for name, g, ref, tol in zip(("dq", "dk", "dv"), grads, refs, tols):
        assert_within(g, ref, tol, name)
    if window > 1:  # (with one visible key dQ and dK are zero but for rounding)
        for name, g, ref in zip(("dq", "dk", "dv"), grads, refs):
            # P, out, dS and the result are rounded, each independently
            assert_close_norm(g, ref, 4 * half_step(dtype), name)
    again = window_attn_bwd(do, q, k, v, out, lse, window, sinks, kv_lens=n)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_large_scores_and_long_rows():
    """Scores far apart: the running maximum moves many times; the last tile walked (the sinks) may hold the largest."""
    from block_sparse_attention import window_attn_fwd
    q, k, v, _ = make(1, 2, 2, 900, 900, 128, BF, seed=3, spread=4.0)
    k[:, :, :4] *= 4.0
    ref, lse, tol, lse_tol, _, _ = attend(q.double(), k.double(), v.double(), masks(1, 900, 900, 400, 4, None), 0.3, BF)
    out, got = window_attn_fwd(q.cuda(), k.cuda(), v.cuda(), 400, 4, softmax_scale=0.3, return_lse=True)
    assert_within(out, ref, tol, "out")
    assert_within(got, lse, lse_tol, "lse")


def test_autograd_strided_and_broadcast_inputs():
    """Views of one fused projection, a KV head broadcast over the batch, and a broadcast output gradient."""
    from block_sparse_attention import window_attention
    B, H, S, D = 2, 4, 260, 64
    g = torch.Generator().manual_seed(5)
    fused = torch.randn(B, S, 3, H, D, generator=g).bfloat16()
    one = torch.randn(1, 2, S, D, generator=g).bfloat16()
    f = fused.cuda().requires_grad_()
    shared = one.cuda().requires_grad_()
    q, k = f[:, :, 0], f[:, :, 1]
    out = window_attention(q, k, f[:, :, 2], 100, 3, layout="bshd")
    kb = shared.expand(B, 2, S, D)
    out2 = window_attention(q.transpose(1, 2), kb, kb, 100, 3)
    (out.float().sum() + 2 * out2.float().sum()).backward()
    fd, od = fused.double(), one.double()
    mask = masks(B, S, S, 100, 3, None)
    tr = lambda t: t.transpose(1, 2)  # noqa: E731
    ones = torch.ones(B, H, S, D, dtype=torch.float64)
    r1, t1 = gradients(tr(fd[:, :, 0]), tr(fd[:, :, 1]), tr(fd[:, :, 2]), ones, mask, D ** -0.5, BF)
    kd = od.expand(B, 2, S, D)
    r2, t2 = gradients(tr(fd[:, :, 0]), kd, kd, 2 * ones, mask, D ** -0.5, BF)
    u = half_step(BF)
    # autograd adds the two uses in bf16: one more rounding of each sum
    want = torch.stack([tr(r1[0] + r2[0]), tr(r1[1]), tr(r1[2])], 2)
    tol = torch.stack([tr(t1[0] + t2[0]), tr(t1[1]), tr(t1[2])], 2) + u * want.abs() * 2
    assert_within(f.grad, want, tol, "fused")
    kv = (r2[1] + r2[2])
    kv_tol = t2[1] + t2[2] + 2 * u * kv.abs()
    assert_within(shared.grad, kv.sum(0, keepdim=True), kv_tol.sum(0, keepdim=True) + 2 * u * kv.abs().sum(0, keepdim=True), "shared")


def test_out_lse_and_gradient_buffers():
    """Buffers of the caller: strided, unaligned, longer than the call; what lies around them is left alone."""
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    q, k, v, do = (t.cuda() for t in make(1, 2, 2, 200, 200, 128, BF, seed=6))
    ref, lse = window_attn_fwd(q, k, v, 60, 2, return_lse=True)
    big = torch.full((1, 2, 300, 128), 7.0, dtype=BF, device="cuda")
    lse_big = torch.full((1, 2, 300), 7.0, device="cuda")
    out, got = window_attn_fwd(q, k, v, 60, 2, out=big[:, :, 50:250], lse=lse_big[:, :, 50:250])
    assert torch.equal(out, ref) and torch.equal(got, lse)
    assert (big[:, :, :50] == 7).all() and (big[:, :, 250:] == 7).all() and (lse_big[:, :, :50] == 7).all()
    odd = torch.zeros(2 * 200 * 128 + 3, dtype=BF, device="cuda")[3:].view(1, 2, 200, 128)
    assert torch.equal(window_attn_fwd(q, k, v, 60, 2, out=odd)[0], ref) and torch.equal(odd, ref)
    shifted = torch.empty(2 * 200 * 128 + 3, dtype=BF, device="cuda")[3:].view(1, 2, 200, 128).copy_(k)
    assert torch.equal(window_attn_fwd(q, shifted, v, 60, 2)[0], ref)
    grads = window_attn_bwd(do, q, k, v, ref, lse, 60, 2)
    hold = [torch.full((1, 2, 300, 128), 7.0, dtype=BF, device="cuda") for _ in range(3)]
    window_attn_bwd(do, q, k, v, ref, lse, 60, 2, dq=hold[0][:, :, 9:209], dk=hold[1][:, :, 9:209], dv=hold[2][:, :, 9:209])
    for h, g in zip(hold, grads):
        assert torch.equal(h[:, :, 9:209], g) and (h[:, :, :9] == 7).all() and (h[:, :, 209:] == 7).all()


def test_empty_extents():
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    out, lse = window_attn_fwd(z(2, 2, 0, 64), z(2, 2, 5, 64), z(2, 2, 5, 64), 4, return_lse=True)
    assert out.shape == (2, 2, 0, 64) and lse.shape == (2, 2, 0)
    q = torch.ones(1, 2, 3, 64, dtype=BF, device="cuda")
    out, lse = window_attn_fwd(q, z(1, 2, 0, 64), z(1, 2, 0, 64), 4, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = window_attn_bwd(q, q, z(1, 2, 0, 64), z(1, 2, 0, 64), out, lse, 4)
    assert (dq == 0).all() and dk.shape == dv.shape == (1, 2, 0, 64)


def test_streams_and_graphs():
    """A side stream, and two captured graphs replayed in turn on new inputs, against direct calls."""
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    sets = [[t.cuda() for t in make(1, 4, 2, 300, 300, 128, BF, seed=s)] for s in range(2)]

    def step(q, k, v, do):
        out, lse = window_attn_fwd(q, k, v, 90, 3, return_lse=True)
        return (out,) + window_attn_bwd(do, q, k, v, out, lse, 90, 3)

    want = [step(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs = []
    for s in sets:
        held = [t.clone() for t in s]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(*held)
        graphs.append((graph, held, res))
    for turn in range(2):
        for i, (graph, held, res) in enumerate(graphs):
            for h, t in zip(held, sets[(i + turn) % 2]):
                h.copy_(t)
            graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, res) in enumerate(graphs):
            assert all(torch.equal(x, y) for x, y in zip(res, want[(i + turn) % 2]))


def test_matches_dense_block_sparse_operator():
    """A window over everything, queries at the end of the keys: the last row equals full attention by the
    block-sparse operator over all blocks (both round P and the result: two half steps each)."""
    from block_sparse_attention import bsa_attn_fwd, window_attn_fwd
    q, k, v, _ = (t.cuda() for t in make(1, 2, 2, 1, 512, 128, BF, seed=8))
    index = torch.arange(4, dtype=torch.int32, device="cuda").expand(1, 2, 1, 4).contiguous()
    a, la = bsa_attn_fwd(q, k, v, index, 4, return_lse=True, sparse_block_size=128)
    b, lb = window_attn_fwd(q, k, v, 512, 0, return_lse=True)
    _, _, tol, lse_tol, _, _ = attend(q.double().cpu(), k.double().cpu(), v.double().cpu(), torch.ones(1, 1, 512, dtype=torch.bool), 128 ** -0.5, BF)
    assert_within(a, b.double().cpu(), 2 * tol, "out")
    assert_within(la, lb.double().cpu(), 2 * lse_tol, "lse")


def test_nan_is_passed_on_to_its_own_row():
    from block_sparse_attention import window_attn_fwd
    for S in (300, 6):  # whole query tiles, and lists cut into runs
        Sk = 300 if S == 300 else 6000
        q, k, v, _ = (t.cuda() for t in make(1, 2, 2, S, Sk, 128, BF, seed=12))
        want, want_lse = window_attn_fwd(q, k, v, 1 << 20, 2, return_lse=True)
        q[0, 1, 3] = float("nan")
        out, lse = window_attn_fwd(q, k, v, 1 << 20, 2, return_lse=True)
        assert out[0, 1, 3].isnan().all() and lse[0, 1, 3].isnan()
        keep = torch.ones(1, 2, S, dtype=torch.bool, device="cuda")
        keep[0, 1, 3] = False
        assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


def test_aliased_buffers_and_second_derivatives_are_refused():
    from block_sparse_attention import window_attention, window_attn_bwd, window_attn_fwd
    q, k, v, do = (t.cuda() for t in make(1, 2, 2, 64, 64, 64, BF))
    out, lse = window_attn_fwd(q, k, v, 9, return_lse=True)
    with pytest.raises(AssertionError):
        window_attn_fwd(q, k, v, 9, out=k)
    with pytest.raises(AssertionError):
        window_attn_bwd(do, q, k, v, out, lse, 9, dq=do)
    both = torch.empty_like(k)
    with pytest.raises(AssertionError):
        window_attn_bwd(do, q, k, v, out, lse, 9, dk=both, dv=both)
    q.requires_grad_()
    g, = torch.autograd.grad(window_attention(q, k, v, 9).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_a_very_long_past():
    """300 000 keys before one query: one list cut over the whole GPU."""
    from block_sparse_attention import window_attn_fwd
    q, k, v, _ = make(1, 2, 1, 1, 300000, 64, BF, seed=13)
    ref, lse, tol, lse_tol, _, _ = attend(q.double(), k.double(), v.double(), torch.ones(1, 1, 300000, dtype=torch.bool), 0.125, BF)
    out, got = window_attn_fwd(q.cuda(), k.cuda(), v.cuda(), 1 << 20, return_lse=True)
    assert_within(out, ref, tol, "out")
    assert_within(got, lse, lse_tol + 2.0 ** -20, "lse")  # (300 000 terms joined from 296 pieces: 2^-22 each of pieces and sum)


def test_two_streams_at_once():
    """Calls that overlap on the GPU: each has its own workspace."""
    from block_sparse_attention import cached_attn_fwd, window_attn_bwd, window_attn_fwd
    sets = [[t.cuda() for t in make(1, 8, 1, 200, 1500, 128, BF, seed=s)] for s in range(2)]
    pools = [torch.randn(40, 1, 64, 128, device="cuda").bfloat16() for _ in range(2)]
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([2500], dtype=torch.int32, device="cuda")

    def step(q, k, v, do):
        out, lse = window_attn_fwd(q, k, v, 1000, 3, return_lse=True)
        return (out, cached_attn_fwd(q, *pools, table, n)[0]) + window_attn_bwd(do, q, k, v, out, lse, 1000, 3)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_another_device_than_the_current_one():
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    a = make(1, 2, 1, 300, 300, 64, BF)
    res = []
    for dev in ("cuda:0", "cuda:1"):
        q, k, v, do = (t.to(dev) for t in a)
        out, lse = window_attn_fwd(q, k, v, 50, 2, return_lse=True)
        res.append([t.cpu() for t in (out,) + window_attn_bwd(do, q, k, v, out, lse, 50, 2)])
    assert all(torch.equal(x, y) for x, y in zip(*res))


@pytest.fixture
def deal(request, monkeypatch):
    """Every call deals its work in the given way, whatever the rule says."""
    from block_sparse_attention import cached_attn, window_attn

    def clear():
        cached_attn._cached_plan.cache_clear()
        window_attn._window_plan.cache_clear()
    monkeypatch.setattr(window_attn, "_deal_work", lambda *sizes: request.param)
    clear()
    yield request.param
    clear()


DEALS = [(0, 1), (0, 2), (0, 5), (0, 8), (1, 1), (7, 1), (296, 1)]


@pytest.mark.parametrize("deal", DEALS, indirect=True, ids=str)
def test_every_way_of_dealing_the_work(deal):
    for case in CASES:
        test_forward(case, "bshd")


GROUPED = [
    (1, 14, 14, 256, 9000, 128, BF, 1 << 20, 2, None),   # ten heads' keys fill the group of the forward and dQ kernels
    (15, 11, 1, 600, 600, 128, BF, 1 << 20, 0, None),    # fourteen heads' queries that of the dK/dV kernel
]


@pytest.mark.parametrize("deal", [(0, 1)], indirect=True, ids=str)
@pytest.mark.parametrize("case", GROUPED, ids=["keys", "queries"])
def test_more_heads_than_are_dealt_at_a_time(deal, case):
    test_forward(case, "bhsd")
    test_backward(case)


def test_captured_training_step():
    """Rotation and attention with their gradients in one captured step, replayed on new inputs, against direct calls."""
    from block_sparse_attention import (rotary_embedding, rotary_frequencies, rotary_nd, window_attention, window_attn_bwd,
                                        window_attn_fwd)
    pairs = (8, 12, 12)
    sets = [[t.cuda() for t in make(2, 6, 2, 333, 333, 64, BF, seed=s)] for s in range(2)]
    q, k, v = (t.clone().requires_grad_() for t in sets[0][:3])
    do = sets[0][3].clone()
    pos = torch.randint(0, 500, (333, 3), generator=torch.Generator().manual_seed(3), dtype=torch.int32).cuda()
    freq = rotary_frequencies(pairs, device="cuda")

    def step():
        a, b = rotary_embedding(q, k, pos, freq, pairs)
        window_attention(a, b, v, 90, 3).backward(do)

    side = torch.cuda.Stream()  # (warmed up there, and the eager graphs dropped, as captures of a backward pass need it)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
            q.grad = k.grad = v.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for new in sets[::-1]:
        with torch.no_grad():
            for held, t in zip((q, k, v, do), new):
                held.copy_(t)
        graph.replay()
        a, b = rotary_nd(new[0], new[1], pos, freq, pairs)
        out, lse = window_attn_fwd(a, b, new[2], 90, 3, return_lse=True)
        da, db, dv = window_attn_bwd(new[3], a, b, new[2], out, lse, 90, 3)
        dq, dk = rotary_nd(da, db, pos, freq, pairs, inverse=True)
        for got, want in zip((q.grad, k.grad, v.grad), (dq, dk, dv)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window,sinks", [(2, 0), (3, 0), (1, 2), (1, 4), (5, 3)])
def test_few_visible_keys_keep_their_gradients(window, sinks, dtype):
    """delta nearly cancels dP there.  dS and the result are each off by at most u / sqrt(3) in the mean square, u half a
    step: together 0.82 u."""
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    lens = [700, 400]
    q, k, v, do = make(2, 6, 2, 600, 700, 128, dtype, seed=5)
    refs, _ = gradients(q.double(), k.double(), v.double(), do.double(), masks(2, 600, 700, window, sinks, lens), 128 ** -0.5, dtype)
    k, v, q, do = poison(k, lens, 0), poison(v, lens, 0), poison(q, lens, 100), poison(do, lens, 100)
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = window_attn_fwd(q, k, v, window, sinks, kv_lens=n, return_lse=True)
    for name, g, ref in zip(("dq", "dk", "dv"), window_attn_bwd(do, q, k, v, out, lse, window, sinks, kv_lens=n), refs):
        assert_close_norm(g, ref, 0.82 * half_step(dtype), name)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Sq,Sk", [(4, 4), (13, 13), (20, 9)])
def test_short_sequences_keep_their_gradients(Sq, Sk, dtype):
    from block_sparse_attention import window_attn_bwd, window_attn_fwd
    q, k, v, do = make(40, 6, 2, Sq, Sk, 64, dtype, seed=6)
    refs, _ = gradients(q.double(), k.double(), v.double(), do.double(), masks(40, Sq, Sk, 100, 3, None), 64 ** -0.5, dtype)
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    out, lse = window_attn_fwd(q, k, v, 100, 3, return_lse=True)
    for name, g, ref in zip(("dq", "dk", "dv"), window_attn_bwd(do, q, k, v, out, lse, 100, 3), refs):
        assert_close_norm(g, ref, 0.82 * half_step(dtype), name)
