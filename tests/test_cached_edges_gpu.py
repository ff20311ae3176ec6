"""GPU parity of cached attention at its edges: short trees, what unseen keys and unused queries hold, lengths and tables, pools."""
import pytest
import torch

from dealing import DEALS, deal  # noqa: F401
from plain_ops import ancestors, assert_within, attend, cached_visible
from test_cached_attn_gpu import ALL, BF, HF, make_cache

pytestmark = pytest.mark.gpu


def tree_visible(T, length, window, sinks, parents):
    """[T, length] bool: a draft's position is base + (drafts on its branch) - 1, also where the branch begins before the
    sequence; drafts whose key would lie before the sequence have none, rows at negative positions see nothing."""
    base = length - T
    chains = ancestors(parents)
    at = [None if c is None else base + len(c) - 1 for c in chains]
    seen = torch.zeros(T, max(length, 0), dtype=torch.bool)
    for t, c in enumerate(chains):
        if c is None or at[t] < 0:
            continue
        keys = [(j, j) for j in range(max(base, 0))] + [(base + u, at[u]) for u in c if base + u >= 0]
        for j, rank in keys:
            seen[t, j] = rank > at[t] - window or rank < sinks
    return seen


def random_tree(T, g):
    return [int(torch.randint(-1, t, (1,), generator=g)) if t else -1 for t in range(T)]


def check(out, lse, q, ks, vs, masks, dtype):
    for b, mask in enumerate(masks):
        ref, rl, tol, lt, _, _ = attend(q[b:b + 1].double(), ks[b][None].double(), vs[b][None].double(), mask[None],
                                        q.shape[-1] ** -0.5, dtype)
        assert_within(out[b:b + 1], ref, tol, f"out of sequence {b}")
        assert_within(lse[b:b + 1], rl, lt, f"lse of sequence {b}")


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


# T, window, sinks, page, Hq, Hkv, D, dtype, lens
SHORT_TREES = [
    (17, 2, 0, 16, 2, 2, 128, BF, [5, 16, 1, 17]),
    (17, 3, 1, 16, 4, 2, 64, HF, [5, 16, 0, 30]),
    (40, 6, 2, 32, 8, 1, 96, BF, [39, 11, 3, 41]),  # several packed query tiles
    (64, None, 0, 64, 2, 1, 64, BF, [63, 20, 1, 64]),
    (64, 4, 3, 128, 6, 2, 96, HF, [63, 20, 2, 700]),
    (33, 1, 0, 384, 2, 2, 64, BF, [32, 500, 7, 33]),
]


@pytest.mark.parametrize("case", SHORT_TREES, ids=[str(i) for i in range(len(SHORT_TREES))])
@pytest.mark.parametrize("shape", ["chain", "random", "star"])
def test_trees_over_sequences_shorter_than_the_tree(case, shape):
    from block_sparse_attention import cached_attn_fwd, tree_mask_from_parents
    T, window, sinks, page, Hq, Hkv, D, dtype, lens = case
    g = torch.Generator().manual_seed(T)
    B = len(lens)
    make = {"chain": lambda: [t - 1 for t in range(T)], "random": lambda: random_tree(T, g), "star": lambda: [-1] + [0] * (T - 1)}
    parents = [make[shape]() for _ in range(B)]
    kc, vc, table, ks, vs = make_cache(B, Hkv, page, D, lens, dtype, seed=T)
    q = torch.randn(B, Hq, T, D, generator=g).to(dtype)
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), i32(lens), tree_mask=tree_mask_from_parents(i32(parents)),
                               window=window, sink_tokens=sinks, return_lse=True)
    check(out, lse, q, ks, vs, [tree_visible(T, n, window or ALL, sinks, p) for n, p in zip(lens, parents)], dtype)


@pytest.mark.parametrize("window,sinks", [(None, 0), (2, 0), (5, 2), (1, 1)])
def test_a_chain_is_a_chunk_of_tokens_also_where_it_begins_before_the_sequence(window, sinks):
    from block_sparse_attention import cached_attn_fwd, tree_mask_from_parents
    lens, T = [5, 29, 1, 0, 30], 30
    kc, vc, table, ks, vs = make_cache(5, 2, 16, 128, lens, BF)
    q = torch.randn(5, 4, T, 128, generator=torch.Generator().manual_seed(2)).bfloat16()
    args = (q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), i32(lens))
    chain = tree_mask_from_parents((torch.arange(T, dtype=torch.int32) - 1).expand(5, T).cuda())
    a = cached_attn_fwd(*args, window=window, sink_tokens=sinks, return_lse=True)
    b = cached_attn_fwd(*args, window=window, sink_tokens=sinks, tree_mask=chain, return_lse=True)
    for got in (a, b):
        check(*got, q, ks, vs, [cached_visible(T, n, window or ALL, sinks) for n in lens], BF)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def poison_unseen(pools, table, masks, holds):
    """Fills the rows of every key in its sequence that no row of its mask sees."""
    page = pools[0].shape[2]
    some = False
    for b, mask in enumerate(masks):
        for j in (~mask.any(0)).nonzero()[:, 0].tolist() if mask.shape[1] else []:
            for pool in pools:
                pool[table[b, j // page], :, j % page] = holds
            some = True
    assert some


# T, window, sinks, page, Hq, Hkv, D, dtype, lens; the trees hold unused slots
UNSEEN = [
    (1, 100, 4, 16, 8, 2, 128, BF, [700, 64, 300]),
    (40, 70, 0, 64, 4, 4, 64, HF, [500, 41]),
    (9, 130, 100, 256, 2, 1, 96, BF, [1000, 300]),
]


@pytest.mark.parametrize("deal", DEALS, indirect=True, ids=str)
@pytest.mark.parametrize("case", UNSEEN, ids=[str(i) for i in range(len(UNSEEN))])
def test_cached_tokens_before_every_window_may_hold_anything(case, deal):
    from block_sparse_attention import cached_attn_fwd
    T, window, sinks, page, Hq, Hkv, D, dtype, lens = case
    kc, vc, table, ks, vs = make_cache(len(lens), Hkv, page, D, lens, dtype, seed=T)
    masks = [cached_visible(T, n, window, sinks) for n in lens]
    poison_unseen((kc, vc), table, masks, float("nan"))
    q = torch.randn(len(lens), Hq, T, D, generator=torch.Generator().manual_seed(T)).to(dtype)
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), i32(lens), window=window, sink_tokens=sinks, return_lse=True)
    check(out, lse, q, ks, vs, masks, dtype)


UNUSED = [
    (20, None, 0, 16, 4, 2, 128, BF, [300, 20, 12, 140]),
    (64, 30, 2, 64, 2, 2, 64, HF, [64, 500, 191, 40]),
    (48, None, 0, 128, 8, 2, 96, BF, [48, 300, 127, 170]),   # two query tiles; drafts on both sides of a key tile's end
    (64, 1, 0, 32, 16, 2, 128, BF, [66, 64, 129, 700]),
]


@pytest.mark.parametrize("deal", DEALS, indirect=True, ids=str)
@pytest.mark.parametrize("case", UNUSED, ids=[str(i) for i in range(len(UNUSED))])
def test_unused_drafts_may_hold_anything(case, deal):
    from block_sparse_attention import cached_attn_fwd, tree_mask_from_parents
    T, window, sinks, page, Hq, Hkv, D, dtype, lens = case
    g = torch.Generator().manual_seed(T)
    parents = [random_tree(T, g) for _ in lens]
    for p in parents:
        for t in (3, 7, T - 1):
            p[t] = -2
    parents[1] = [-2] * T  # no draft at all
    kc, vc, table, ks, vs = make_cache(len(lens), Hkv, page, D, lens, dtype, seed=T)
    masks = [tree_visible(T, n, window or ALL, sinks, p) for n, p in zip(lens, parents)]
    poison_unseen((kc, vc), table, masks, float("nan"))
    q = torch.randn(len(lens), Hq, T, D, generator=g).to(dtype)
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), i32(lens), tree_mask=tree_mask_from_parents(i32(parents)),
                               window=window, sink_tokens=sinks, return_lse=True)
    check(out, lse, q, ks, vs, masks, dtype)


@pytest.mark.parametrize("beyond", [1, 5, 40, 2 ** 31 - 1 - 96])
def test_a_length_beyond_the_table_is_the_table_in_every_call(beyond):
    """Write, attend, keep: what the calls do for the table's own length."""
    from block_sparse_attention import cache_append, cache_keep, cached_attn_fwd
    T, full = 5, 96
    g = torch.Generator().manual_seed(8)
    kc, vc, table, _, _ = make_cache(2, 2, 32, 64, [full, full], BF, garbage=False)
    q, k, v = (torch.randn(2, h, T, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2))
    path = i32([[0, 2, 4], [1, 3, 4]])

    def step(n):
        pools = kc.clone().cuda(), vc.clone().cuda()
        cache_append(k, v, *pools, table.cuda(), i32(n))
        out, lse = cached_attn_fwd(q, *pools, table.cuda(), i32(n), window=40, return_lse=True)
        new = cache_keep(*pools, table.cuda(), i32(n), path, i32([3, 2]), T)
        return (out, lse, new) + pools

    want = step([full, full])
    assert torch.equal(want[2], i32([full - 2, full - 3])) and not torch.equal(want[3].cpu(), kc)
    assert all(torch.equal(a, b) for a, b in zip(step([full + beyond, full]), want))


def test_a_window_over_the_longest_table():
    """2^29 places a sequence, of which a window sees a few: the list of key tiles is that of the windows."""
    from block_sparse_attention import cached_attn_fwd
    from block_sparse_attention.window_attn import _deal_work
    B, page, n = 607, 1 << 20, 5000
    assert _deal_work(B, 18, 1, False, 148)[0] > 0  # shared evenly, as the call below
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(1, 1, n, 64, generator=g).bfloat16() for _ in range(2))
    pools = [torch.zeros(1, 1, page, 64, dtype=BF, device="cuda") for _ in range(2)]
    for pool, x in zip(pools, (k, v)):
        pool[:, :, :n] = x.cuda()
    table = torch.zeros(B, 512, dtype=torch.int32, device="cuda")
    q = torch.randn(1, 1, 1, 64, generator=g).bfloat16()
    out, lse = cached_attn_fwd(q.cuda().expand(B, 1, 1, 64).contiguous(), *pools, table, i32([n] * B), window=2000, return_lse=True)
    check(out[::150], lse[::150], q.expand(5, 1, 1, 64), [k[0]] * 5, [v[0]] * 5, [cached_visible(1, n, 2000, 0)] * 5, BF)


@pytest.mark.parametrize("deal", DEALS, indirect=True, ids=str)
def test_results_do_not_depend_on_unused_queries(deal):
    """To the bit: queries of unused slots and of tokens before the sequence."""
    from block_sparse_attention import cached_attn_fwd, tree_mask_from_parents
    lens, T = [900, 20, 300], 40
    kc, vc, table, _, _ = make_cache(3, 2, 64, 128, lens, BF)
    g = torch.Generator().manual_seed(10)
    q = torch.randn(3, 4, T, 128, generator=g).bfloat16()
    parents = [[-1 if t % 7 == 0 else -2 if t % 7 == 3 else t - 1 for t in range(T)] for _ in lens]
    mask = tree_mask_from_parents(i32(parents))
    unused = (mask == 0).cpu()[:, None, :, None]
    before = (torch.arange(T) + torch.tensor(lens)[:, None] < T)[:, None, :, None]
    assert unused.any() and before.any()
    pools = kc.cuda(), vc.cuda(), table.cuda(), i32(lens)
    for dead, tree in ((unused | before, mask), (before, None)):
        got = []
        for holds in (1.0, 30.0, -1000.0, float("nan")):
            got.append(cached_attn_fwd(torch.where(dead, q * holds, q).cuda(), *pools, tree_mask=tree, return_lse=True))
        for other in got[1:]:
            assert torch.equal(got[0][0], other[0]) and torch.equal(got[0][1], other[1])


def test_pools_that_interleave_are_written():
    from block_sparse_attention import cache_append, cache_keep
    kc, vc, table, _, _ = make_cache(2, 2, 16, 64, [50, 40], BF, garbage=False)
    both = torch.stack((kc, vc), 1).cuda()
    rows = torch.stack([torch.randn(2, 2, 9, 64, generator=torch.Generator().manual_seed(s)).bfloat16() for s in (1, 2)], 2).cuda()
    k, v = rows[:, :, 0], rows[:, :, 1]
    kc, vc, table, n = kc.cuda(), vc.cuda(), table.cuda(), i32([50, 40])
    path, counts = i32([[1, 4, 8], [0, 2, 3]]), i32([3, 2])
    for pools in ((kc, vc), (both[:, 0], both[:, 1])):
        cache_append(k, v, *pools, table, n)
        new = cache_keep(*pools, table, n, path, counts, 9)
        assert new.tolist() == [44, 33]
    assert torch.equal(both[:, 0], kc) and torch.equal(both[:, 1], vc)


@pytest.mark.parametrize("deal", DEALS[1:], indirect=True, ids=str)
def test_every_way_of_dealing_short_trees(deal):
    for case in SHORT_TREES:
        test_trees_over_sequences_shorter_than_the_tree(case, "random")


# Hq, Hkv, T, page, D, dtype, lens, window, sinks
CHUNKS = [
    (4, 2, 600, 384, 64, HF, [1500, 640], None, 0),       # pages of three key tiles
    (8, 1, 300, 64, 96, BF, [2000, 300, 299], 500, 4),
    (2, 2, 1024, 16, 128, BF, [1024], 129, 1),
    (32, 8, 512, 128, 128, BF, [4096], None, 0),
]


@pytest.mark.parametrize("case", CHUNKS, ids=[str(i) for i in range(len(CHUNKS))])
def test_chunks_of_a_prompt(case):
    from block_sparse_attention import cached_attn_fwd
    Hq, Hkv, T, page, D, dtype, lens, window, sinks = case
    kc, vc, table, ks, vs = make_cache(len(lens), Hkv, page, D, lens, dtype, seed=T)
    q = torch.randn(len(lens), Hq, T, D, generator=torch.Generator().manual_seed(T)).to(dtype)
    out, lse = cached_attn_fwd(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), i32(lens), window=window, sink_tokens=sinks, return_lse=True)
    p = [torch.arange(n - T, n)[:, None] for n in lens]
    masks = [(torch.arange(n) <= x) & ((torch.arange(n) > x - (window or ALL)) | (torch.arange(n) < sinks)) & (x >= 0)
             for n, x in zip(lens, p)]
    check(out, lse, q, ks, vs, masks, dtype)


def test_a_table_without_pages_holds_no_token():
    from block_sparse_attention import cache_append, cache_keep, cached_attn_fwd
    pools = [torch.ones(3, 2, 16, 64, dtype=BF, device="cuda") for _ in range(2)]
    x, table, n = torch.ones(2, 2, 4, 64, dtype=BF, device="cuda"), torch.empty(2, 0, dtype=torch.int32, device="cuda"), i32([9, 0])
    cache_append(2 * x, 2 * x, *pools, table, n)
    new = cache_keep(*pools, table, n, i32([[1, 2], [0, 1]]), i32([2, 2]), 4)
    out, lse = cached_attn_fwd(x, *pools, table, n, return_lse=True)
    assert torch.equal(new, n) and new.data_ptr() != n.data_ptr()  # fewer tokens than drafts: left as they are
    assert all((p == 1).all() for p in pools) and (out == 0).all() and lse.isneginf().all()
