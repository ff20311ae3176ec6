"""GPU parity of attention over a paged cache (single tokens, chunks, trees of drafts) and of the cache's writes."""
import math

import pytest
import torch

from plain_ops import assert_within, attend, cached_visible

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
ALL = 1 << 29


def make_cache(B, Hkv, page, D, lens, dtype, seed=0, extra=3, garbage=True):
    """Pools whose pages are dealt at random; what no sequence owns, and the ends of last pages, hold NaN."""
    g = torch.Generator().manual_seed(seed)
    most = max(1, max(-(-n // page) for n in lens))
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(need) + extra, generator=g)
    pools = [torch.full((len(ids), Hkv, page, D), float("nan") if garbage else 0.0, dtype=dtype) for _ in range(2)]
    table = torch.full((B, most), -1, dtype=torch.int32)
    dense = [[], []]
    at = 0
    for b, n in enumerate(lens):
        mine = ids[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = mine.to(torch.int32)
        for c in range(2):
            x = torch.randn(Hkv, n, D, generator=g).to(dtype)
            dense[c].append(x)
            for s, page_id in enumerate(mine.tolist()):
                part = x[:, s * page:(s + 1) * page]
                pools[c][page_id, :, :part.shape[1]] = part
    return pools[0], pools[1], table, dense[0], dense[1]


def check(out, lse, q, ks, vs, lens, window, sinks, scale, dtype, parents=None, lost=None):
    """lost[b]: positions of sequence b whose page is gone."""
    for b, n in enumerate(lens):
        T = q.shape[2]
        mask = cached_visible(T, n, window, sinks, None if parents is None else parents[b])
        if lost is not None and lost[b]:
            mask[:, lost[b]] = False
        ref, rl, tol, lt, _, _ = attend(q[b:b + 1].double(), ks[b][None].double(), vs[b][None].double(), mask[None], scale, dtype)
        assert_within(out[b:b + 1], ref, tol, f"out of sequence {b}")
        assert_within(lse[b:b + 1], rl, lt, f"lse of sequence {b}")


# Hq, Hkv, T, page, D, dtype, lens, window, sinks
CASES = [
    (4, 4, 1, 16, 128, BF, [1], None, 0),
    (8, 2, 1, 16, 128, BF, [5, 300, 1, 129, 0], None, 0),
    (8, 1, 1, 64, 64, HF, [1000, 64, 65], 200, 4),
    (3, 1, 1, 32, 96, BF, [127, 128, 129], 64, 1),
    (6, 2, 7, 16, 128, HF, [200, 7, 3, 95], 50, 2),     # a sequence with fewer tokens than the chunk
    (2, 2, 130, 128, 128, BF, [130, 700], 140, 100),
    (16, 2, 40, 256, 128, BF, [900, 41], None, 0),       # five packed tiles
    (4, 4, 3, 64, 64, BF, [3000], 700, 128),             # keys split over many CTAs
    (10, 2, 2, 128, 128, HF, [1500, 20], 1, 5),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_tokens(case, layout):
    from block_sparse_attention import cached_attn_fwd
    Hq, Hkv, T, page, D, dtype, lens, window, sinks = case
    kc, vc, table, ks, vs = make_cache(len(lens), Hkv, page, D, lens, dtype)
    q = torch.randn(len(lens), Hq, T, D, generator=torch.Generator().manual_seed(9)).to(dtype)
    qd = q.cuda() if layout == "bhsd" else q.transpose(1, 2).contiguous().cuda()
    out, lse = cached_attn_fwd(qd, kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                               window=window, sink_tokens=sinks, return_lse=True, layout=layout)
    out = out if layout == "bhsd" else out.transpose(1, 2)
    check(out, lse, q, ks, vs, lens, window or ALL, sinks, D ** -0.5, dtype)


TREES = [
    # T, window, sinks, page, Hq, Hkv, lens
    (1, None, 0, 16, 4, 2, [1, 40]),
    (13, None, 0, 16, 4, 4, [13, 300, 140]),
    (64, None, 0, 64, 8, 2, [64, 700, 127, 191]),
    (64, 100, 4, 32, 2, 1, [64, 500]),
    (33, 3, 2, 128, 6, 2, [33, 260, 40]),   # a window shorter than the branches
    (20, 1, 0, 16, 2, 2, [25, 20]),
    (17, None, 0, 16, 2, 2, [5, 0, 17]),    # fewer tokens than drafts
]


@pytest.mark.parametrize("tree", TREES, ids=[str(i) for i in range(len(TREES))])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_trees(tree, dtype):
    from block_sparse_attention import cached_attn_fwd, tree_mask_from_parents
    T, window, sinks, page, Hq, Hkv, lens = tree
    g = torch.Generator().manual_seed(T)
    B = len(lens)
    parents = [[int(torch.randint(-1, t, (1,), generator=g)) if t else -1 for t in range(T)] for _ in range(B)]
    parents[0] = [t - 1 for t in range(T)]  # a chain
    if T > 10:
        parents[-1][7] = -2  # an unused slot, and whatever hangs from it
        parents[-1][9] = 20  # a parent that comes later
    kc, vc, table, ks, vs = make_cache(B, Hkv, page, 128, lens, dtype, seed=T)
    q = torch.randn(B, Hq, T, 128, generator=g).to(dtype)
    mask = tree_mask_from_parents(torch.tensor(parents, dtype=torch.int32).cuda())
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                               tree_mask=mask, window=window, sink_tokens=sinks, return_lse=True)
    check(out, lse, q, ks, vs, lens, window or ALL, sinks, 128 ** -0.5, dtype, parents)
    # unused bits of a mask (drafts from T on) are ignored
    if T < 64:
        out2, _ = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                  tree_mask=torch.where(mask != 0, mask | (1 << T), mask), window=window, sink_tokens=sinks)
        assert torch.equal(out, out2)


def test_chain_equals_tokens():
    """A tree that is a chain is a chunk of tokens."""
    from block_sparse_attention import cached_attn_fwd, tree_mask_from_parents
    lens = [200, 33, 64]
    kc, vc, table, _, _ = make_cache(3, 2, 16, 128, lens, BF)
    q = torch.randn(3, 4, 30, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    args = (q, kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    chain = tree_mask_from_parents((torch.arange(30, dtype=torch.int32) - 1).expand(3, 30).cuda())
    for window in (None, 20):
        a = cached_attn_fwd(*args, window=window, sink_tokens=3, return_lse=True)
        b = cached_attn_fwd(*args, window=window, sink_tokens=3, tree_mask=chain, return_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_bad_pages():
    """Table entries outside the pool: their tokens are not visible; lengths beyond the table are cut to it."""
    from block_sparse_attention import cached_attn_fwd
    lens = [300, 300]
    kc, vc, table, ks, vs = make_cache(2, 2, 32, 64, lens, BF)
    table[0, 3] = -7
    table[0, 9] = kc.shape[0]
    table[1, 0] = 2 ** 31 - 1
    q = torch.randn(2, 4, 2, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    lost = [list(range(96, 128)) + list(range(288, 300)), list(range(32))]
    check(out, lse, q, ks, vs, lens, ALL, 0, 64 ** -0.5, BF, lost=lost)
    table[:] = -1
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    kc, vc, table, ks, vs = make_cache(1, 2, 32, 64, [64], BF)
    out, lse = cached_attn_fwd(q[:1].cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor([1000], dtype=torch.int32).cuda(), return_lse=True)
    check(out, lse, q[:1], ks, vs, [64], ALL, 0, 64 ** -0.5, BF)


def test_same_pages_in_two_sequences_and_other_layouts():
    """A shared prefix (the same pages in several tables), and pools that store tokens before heads."""
    from block_sparse_attention import cached_attn_fwd
    kc, vc, table, ks, vs = make_cache(1, 2, 16, 128, [200], BF)
    table = table.expand(3, -1).contiguous()
    lens = [200, 150, 17]
    q = torch.randn(3, 8, 1, 128, generator=torch.Generator().manual_seed(2)).bfloat16()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n, return_lse=True)
    check(out, lse, q, [ks[0][:, :m] for m in lens], [vs[0][:, :m] for m in lens], lens, ALL, 0, 128 ** -0.5, BF)
    nhd = [p.transpose(1, 2).contiguous().cuda().transpose(1, 2) for p in (kc, vc)]
    both = torch.stack([kc, vc], 1).cuda()  # one pool of K and V pages
    assert torch.equal(cached_attn_fwd(q.cuda(), *nhd, table.cuda(), n)[0], out)
    assert torch.equal(cached_attn_fwd(q.cuda(), both[:, 0], both[:, 1], table.cuda(), n)[0], out)


def test_far_pages_of_a_large_pool():
    """Page offsets beyond 2^31 elements."""
    from block_sparse_attention import cache_append, cached_attn_fwd
    pages = (1 << 31) // (128 * 64) + 9
    kc = torch.zeros(pages, 1, 128, 64, dtype=BF, device="cuda")
    vc = torch.zeros(pages, 1, 128, 64, dtype=BF, device="cuda")
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, 1, 300, 64, generator=g).bfloat16() for _ in range(2))
    n = torch.tensor([300], dtype=torch.int32, device="cuda")
    cache_append(k.cuda(), v.cuda(), kc, vc, table, n)
    assert torch.equal(kc[pages - 1, 0].cpu(), k[0, 0, :128]) and torch.equal(vc[pages - 2, 0, :44].cpu(), v[0, 0, 256:])
    q = torch.randn(1, 2, 1, 64, generator=g).bfloat16()
    out, lse = cached_attn_fwd(q.cuda(), kc, vc, table, n, return_lse=True)
    check(out, lse, q, [k[0]], [v[0]], [300], ALL, 0, 64 ** -0.5, BF)


@pytest.mark.parametrize("page,T,D,layout", [(16, 1, 128, "bhsd"), (5, 9, 64, "bshd"), (64, 70, 96, "bhsd"), (256, 33, 8, "bshd")])
def test_append(page, T, D, layout):
    from block_sparse_attention import cache_append
    lens = [T, T + 50, 3, 0, 2 * T + 7]
    kc, vc, table, _, _ = make_cache(len(lens), 3, page, D, lens, HF, garbage=False)
    table[4, 0] = 10 ** 6  # not in the pool
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(len(lens), 3, T, D, generator=g).half() for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    for b, n in enumerate(lens):
        for t in range(T):
            pos = n - T + t
            if pos >= 0 and 0 <= table[b, pos // page] < kc.shape[0]:
                want_k[table[b, pos // page], :, pos % page] = k[b, :, t]
                want_v[table[b, pos // page], :, pos % page] = v[b, :, t]
    kc, vc = kc.cuda(), vc.cuda()
    put = (lambda t: t.cuda()) if layout == "bhsd" else (lambda t: t.transpose(1, 2).contiguous().cuda())
    got = cache_append(put(k), put(v), kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), layout=layout)
    assert got[0] is kc and got[1] is vc
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)


def test_one_pool_for_keys_and_values_is_not_written():
    from block_sparse_attention import cache_append, cache_keep
    pool = torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda")
    table, lens = torch.tensor([[0]], dtype=torch.int32).cuda(), torch.tensor([3], dtype=torch.int32).cuda()
    rows = torch.ones(1, 2, 3, 64, dtype=BF, device="cuda")
    with pytest.raises(AssertionError):
        cache_append(rows, rows, pool, pool, table, lens)
    with pytest.raises(AssertionError):
        cache_keep(pool, pool, table, lens, table, lens, 3)
    assert not pool.any()


def test_append_from_strided_and_broadcast_rows():
    from block_sparse_attention import cache_append
    kc, vc, table, _, _ = make_cache(2, 2, 16, 64, [20, 20], BF, garbage=False)
    kc, vc = kc.cuda(), vc.cuda()
    n = torch.tensor([20, 20], dtype=torch.int32).cuda()
    wide = torch.randn(2, 20, 2, 3, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    k = wide[:, :, :, 0].transpose(1, 2)
    v = torch.randn(1, 2, 20, 67, device="cuda").bfloat16()[..., 3:].expand(2, 2, 20, 64)  # rows on odd addresses
    cache_append(k, v, kc, vc, table.cuda(), n)
    for b in range(2):
        for pos in range(20):
            page = int(table[b, pos // 16])
            assert torch.equal(kc[page, :, pos % 16], k[b, :, pos]) and torch.equal(vc[page, :, pos % 16], v[b, :, pos])


def test_keep():
    from block_sparse_attention import cache_keep
    T, page = 24, 16
    lens = [T, 100, 61, 10, 0, 77]
    paths = [[0, 1, 2], [3, 5, 6, 11, 12, 13, 14, 20, 21, 22, 23], [], [1, 2], [0], [4, 9, 9, 12]]
    counts = [3, 11, 0, 2, 1, 4]
    kept = [3, 11, 0, None, None, 2]  # None: fewer tokens than drafts; an entry that does not ascend ends the path
    kc, vc, table, ks, vs = make_cache(len(lens), 2, page, 64, lens, BF, garbage=False)
    path = torch.full((len(lens), 11), 99, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    want_k, want_v = kc.clone(), vc.clone()
    for b, n in enumerate(lens):
        for i in range(kept[b] or 0):
            src, dst = n - T + paths[b][i], n - T + i
            for pool, old in ((want_k, kc), (want_v, vc)):
                pool[table[b, dst // page], :, dst % page] = old[table[b, src // page], :, src % page]
    kc, vc = kc.cuda(), vc.cuda()
    args = (table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    new = cache_keep(kc, vc, *args, path.cuda(), torch.tensor(counts, dtype=torch.int32).cuda(), T)
    assert new.tolist() == [n if m is None else n - T + m for n, m in zip(lens, kept)]
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)
    # counts beyond the path's width, and a move from a page that is gone
    new = cache_keep(kc, vc, *args, path[:, :2].contiguous().cuda(), torch.tensor([9] * 6, dtype=torch.int32).cuda(), T)
    assert new.tolist()[:2] == [lens[0] - T + 2, lens[1] - T + 2]
    none = torch.full_like(table, -1).cuda()
    before = kc.clone()
    cache_keep(kc, vc, none, args[1], path.cuda(), torch.tensor(counts, dtype=torch.int32).cuda(), T)
    assert torch.equal(kc, before)


def test_decoding_run():
    """Rotation, append, window attention as a prefill, tree verification, compaction, the next token: as in use."""
    from block_sparse_attention import (cache_append, cache_keep, cached_attn_fwd, rotary_frequencies, rotary_nd,
                                        tree_mask_from_parents, window_attn_fwd)
    g = torch.Generator().manual_seed(11)
    Hq, Hkv, D, page, S, T = 4, 2, 64, 16, 150, 12
    window, sinks, pairs = 70, 4, (8, 12, 12)
    freq = rotary_frequencies(pairs, device="cuda")
    rnd = lambda h, n: torch.randn(1, h, n, D, generator=g).bfloat16().cuda()  # noqa: E731
    at = lambda p: p.to(torch.int32)[:, None].expand(-1, 3).contiguous().cuda()  # noqa: E731
    kc = torch.full((40, Hkv, page, D), float("nan"), dtype=BF, device="cuda")
    vc = kc.clone()
    table = torch.randperm(40, generator=g)[:20].to(torch.int32)[None].cuda()
    lens = lambda n: torch.tensor([n], dtype=torch.int32).cuda()  # noqa: E731
    q, k, v = rnd(Hq, S), rnd(Hkv, S), rnd(Hkv, S)
    q, k = rotary_nd(q, k, at(torch.arange(S)), freq, pairs)
    cache_append(k, v, kc, vc, table, lens(S))
    prefill, _ = window_attn_fwd(q, k, v, window, sinks)
    over_cache, _ = cached_attn_fwd(q, kc, vc, table, lens(S), window=window, sink_tokens=sinks)
    mask = torch.stack([cached_visible(S, S, window, sinks)])
    ref, _, tol, _, _, _ = attend(q.double().cpu(), k.double().cpu(), v.double().cpu(), mask, D ** -0.5, BF)
    assert_within(prefill, ref, tol, "prefill")
    assert_within(over_cache, ref, tol, "prefill over the cache")
    parents = [-1, 0, 0, 1, 3, 2, 4, 6, 5, 7, 9, 9]
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    dq, dk, dv = rnd(Hq, T), rnd(Hkv, T), rnd(Hkv, T)
    dq, dk = rotary_nd(dq, dk, at(S + torch.tensor(depth)), freq, pairs)
    cache_append(dk, dv, kc, vc, table, lens(S + T))
    tree = tree_mask_from_parents(torch.tensor([parents], dtype=torch.int32).cuda())
    out, lse = cached_attn_fwd(dq, kc, vc, table, lens(S + T), tree_mask=tree, window=window, sink_tokens=sinks, return_lse=True)
    ka, va = torch.cat((k, dk), 2)[0].cpu(), torch.cat((v, dv), 2)[0].cpu()
    check(out, lse, dq.cpu(), [ka], [va], [S + T], window, sinks, D ** -0.5, BF, [parents])
    path = [0, 1, 3, 4, 6]
    new = cache_keep(kc, vc, table, lens(S + T), torch.tensor([path], dtype=torch.int32).cuda(), lens(len(path)), T)
    assert new.tolist() == [S + len(path)]
    tq, tk, tv = rnd(Hq, 1), rnd(Hkv, 1), rnd(Hkv, 1)
    tq, tk = rotary_nd(tq, tk, at(S + len(path) + torch.arange(1)), freq, pairs)
    cache_append(tk, tv, kc, vc, table, new + 1)
    out, lse = cached_attn_fwd(tq, kc, vc, table, new + 1, window=window, sink_tokens=sinks, return_lse=True)
    sel = torch.tensor(path)
    ka = torch.cat((k.cpu(), dk.cpu()[:, :, sel], tk.cpu()), 2)[0]
    va = torch.cat((v.cpu(), dv.cpu()[:, :, sel], tv.cpu()), 2)[0]
    check(out, lse, tq.cpu(), [ka], [va], [S + len(path) + 1], window, sinks, D ** -0.5, BF)


def test_graph_of_a_decoding_step():
    """One captured step, replayed while lengths, tables and tokens change in place, against direct calls."""
    from block_sparse_attention import cache_append, cached_attn_fwd
    lens = [90, 200, 5]
    kc, vc, table, _, _ = make_cache(3, 2, 16, 128, [260, 260, 260], BF, garbage=False)
    kc, vc, table = kc.cuda(), vc.cuda(), table.cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(3, h, 1, 128, generator=g).bfloat16().cuda() for h in (8, 2, 2))

    def step():
        cache_append(k, v, kc, vc, table, n)
        return cached_attn_fwd(q, kc, vc, table, n, window=100, sink_tokens=2)[0]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for turn in range(3):
        n += 17
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        graph.replay()
        got = res.clone()
        assert torch.equal(got, step())


def test_negative_lengths_are_empty_sequences():
    from block_sparse_attention import cache_append, cache_keep, cached_attn_fwd
    kc, vc, table, _, _ = make_cache(2, 2, 16, 64, [40, 40], BF, garbage=False)
    kc, vc, table = kc.cuda(), vc.cuda(), table.cuda()
    n = torch.tensor([-5, -2 ** 31], dtype=torch.int32, device="cuda")
    x = torch.ones(2, 2, 3, 64, dtype=BF, device="cuda")
    before = kc.clone()
    cache_append(x, x, kc, vc, table, n)
    path = torch.tensor([[1], [1]], dtype=torch.int32, device="cuda")
    new = cache_keep(kc, vc, table, n, path, torch.ones(2, dtype=torch.int32, device="cuda"), 3)
    assert torch.equal(kc, before) and torch.equal(new, n)
    out, lse = cached_attn_fwd(x, kc, vc, table, n, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_strided_metadata_of_a_single_sequence():
    """Row views whose strides are those of a larger table."""
    from block_sparse_attention import cached_attn_fwd
    kc, vc, table, ks, vs = make_cache(1, 2, 16, 64, [100], BF)
    wide = torch.full((3, 20), -1, dtype=torch.int32)
    wide[1, :7] = table[0]
    lens = torch.tensor([1, 2, 100, 4], dtype=torch.int32)
    q = torch.randn(1, 4, 1, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    for t, n in ((wide.cuda()[1:2], lens.cuda()[2:3]), (wide.cuda()[1:2, :7], lens.cuda()[2::2][:1])):
        out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), t, n, return_lse=True)
        check(out, lse, q, ks, vs, [100], ALL, 0, 64 ** -0.5, BF)
    cols = wide.cuda().t().contiguous().t()[1:2, :7]  # columns far apart
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), cols, lens.cuda()[2:3], return_lse=True)
    check(out, lse, q, ks, vs, [100], ALL, 0, 64 ** -0.5, BF)


def test_many_ragged_sequences():
    """More sequences than a warp has lanes, lists of very different lengths cut into equal runs."""
    from block_sparse_attention import cached_attn_fwd
    g = torch.Generator().manual_seed(21)
    lens = [int(x) for x in torch.randint(0, 2500, (70,), generator=g)]
    lens[3] = 0
    kc, vc, table, ks, vs = make_cache(70, 1, 64, 64, lens, BF)
    q = torch.randn(70, 2, 1, 64, generator=g).bfloat16()
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    check(out, lse, q, ks, vs, lens, ALL, 0, 64 ** -0.5, BF)


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
    """More CTAs in a team than key tiles, runs that end anywhere, more CTAs than there is work."""
    for case in CASES:
        test_tokens(case, "bhsd")
    for tree in TREES:
        test_trees(tree, BF)
