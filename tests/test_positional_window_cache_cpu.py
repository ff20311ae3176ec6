"""CPU: refusals of the windowed, cached and positional operators, their C entry points' argument checks, struct layouts,
the split rule, and the 64-bit gradient formula that the GPU tests use (against differences)."""
import ctypes
import os
import re

import pytest
import torch

from plain_ops import attend, gradients, visible

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header():
    from block_sparse_attention import _cabi
    text = open(os.path.join(ROOT, "include", "bsa_b200.h")).read()
    for struct, cls in (("bsa_window_fwd_args", _cabi.WindowFwdArgs), ("bsa_window_bwd_args", _cabi.WindowBwdArgs),
                        ("bsa_rotary_args", _cabi.RotaryArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, flags=re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            decl = re.sub(r"^(const\s+)?\w+\s+", "", re.sub(r"\*", " ", decl))
            names += [re.sub(r"\[.*\]", "", n).strip() for n in decl.split(",")]
        assert names == [f[0] for f in cls._fields_], struct


def test_python_refusals():
    import block_sparse_attention as bsa
    q = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    lse = torch.zeros(1, 2, 8)
    i32 = torch.zeros(1, 1, dtype=torch.int32)
    for bad in ((0, 0), (1.5, 0), (True, 0), (4, -1), (4, 129), (4, 1.0)):
        with pytest.raises(AssertionError):
            bsa.window_attn_fwd(q, q, q, *bad)
        with pytest.raises(AssertionError):
            bsa.window_attn_bwd(q, q, q, q, q, lse, *bad)
    for call in (lambda: bsa.window_attn_fwd(q, q, q, 4),  # CPU tensors, everywhere
                 lambda: bsa.window_attention(q, q, q, 4),
                 lambda: bsa.window_attn_bwd(q, q, q, q, q, lse, 4),
                 lambda: bsa.window_attn_fwd(q, q, q, 4, layout="sbhd"),
                 lambda: bsa.cached_attn_fwd(q, q, q, i32, i32[0]),
                 lambda: bsa.cache_append(q, q, q, q, i32, i32[0]),
                 lambda: bsa.cache_keep(q, q, i32, i32[0], i32, i32[0], 1),
                 lambda: bsa.tree_mask_from_parents(i32),
                 lambda: bsa.rotary_nd(q, q, torch.zeros(8, 1, dtype=torch.int32), torch.ones(32), (32,))):
        with pytest.raises(AssertionError):
            call()
    assert bsa.rotary_frequencies((2, 3)).shape == (5,)
    torch.testing.assert_close(bsa.rotary_frequencies((2, 2), theta=16.0), torch.tensor([1.0, 0.25, 1.0, 0.25]))
    torch.testing.assert_close(bsa.rotary_frequencies((2, 2), theta=16.0, shared_ladder=True), torch.tensor([1.0, 0.5, 0.25, 0.125]))


class _FakeCuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: reaches the checks behind the device check."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    is_cuda = property(lambda self: True)


def test_python_refusals_behind_the_device_check():
    import block_sparse_attention as bsa
    f = lambda *s, dt=torch.bfloat16: _FakeCuda(torch.zeros(*s, dtype=dt))  # noqa: E731
    i = lambda *s: _FakeCuda(torch.zeros(*s, dtype=torch.int32))  # noqa: E731
    q = f(2, 4, 8, 64)
    calls = [
        lambda: bsa.window_attn_fwd(f(2, 4, 8, 80), f(2, 4, 8, 80), f(2, 4, 8, 80), 4),     # head dimension
        lambda: bsa.window_attn_fwd(q, f(2, 3, 8, 64), f(2, 3, 8, 64), 4),                   # 4 heads on 3
        lambda: bsa.window_attn_fwd(q, f(1, 4, 8, 64), f(1, 4, 8, 64), 4),                   # batch
        lambda: bsa.window_attn_fwd(q, q, f(2, 4, 9, 64), 4),
        lambda: bsa.window_attn_fwd(q, q, f(2, 4, 8, 64, dt=torch.float16), 4),
        lambda: bsa.window_attn_fwd(f(2, 4, 8, 64, dt=torch.float32), f(2, 4, 8, 64, dt=torch.float32), f(2, 4, 8, 64, dt=torch.float32), 4),
        lambda: bsa.window_attn_fwd(q, q, q, 4, kv_lens=i(3)),
        lambda: bsa.window_attn_fwd(q, q, q, 4, kv_lens=f(2)),
        lambda: bsa.window_attn_fwd(q, q, q, 4, softmax_scale=0.0),
        lambda: bsa.window_attn_fwd(q, q, q, 4, softmax_scale=float("inf")),
        lambda: bsa.window_attn_fwd(q, q, q, 4, out=f(2, 4, 9, 64)),
        lambda: bsa.window_attn_fwd(q, q, q, 4, lse=f(2, 4, 8)),
        lambda: bsa.window_attn_bwd(q, q, q, q, f(2, 4, 9, 64), f(2, 4, 8, dt=torch.float32), 4),
        lambda: bsa.window_attn_bwd(q, q, q, q, q, f(2, 4, 9, dt=torch.float32), 4),
        lambda: bsa.window_attn_bwd(q, q, q, q, q, f(2, 4, 8, dt=torch.float32), 4, dk=f(2, 4, 9, 64)),
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 24, 64), f(3, 4, 24, 64), i(2, 3), i(2)),       # page size
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 128), f(3, 4, 16, 128), i(2, 3), i(2)),     # head dimension
        lambda: bsa.cached_attn_fwd(q, f(3, 3, 16, 64), f(3, 3, 16, 64), i(2, 3), i(2)),       # heads
        lambda: bsa.cached_attn_fwd(q, f(0, 4, 16, 64), f(0, 4, 16, 64), i(2, 3), i(2)),       # no pages
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 64), f(3, 4, 16, 64), i(1, 3), i(2)),
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), None),
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2), window=0),
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2), tree_mask=i(2, 8)),
        lambda: bsa.cached_attn_fwd(f(2, 4, 65, 64), f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2), tree_mask=f(2, 65, dt=torch.int64)),
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 72)[..., :64], f(3, 4, 16, 72)[..., 8:], i(2, 3), i(2, 1)),
        lambda: bsa.cached_attn_fwd(q, f(3, 4, 16, 65)[..., :64], f(3, 4, 16, 65)[..., :64], i(2, 3), i(2)),  # rows of 130 bytes
        lambda: bsa.cached_attn_fwd(q, f(1, 4, 16, 64).expand(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2)),
        lambda: bsa.tree_mask_from_parents(i(2, 65)),
        lambda: bsa.cache_append(q, q, f(3, 4, 16, 64, dt=torch.float16), f(3, 4, 16, 64, dt=torch.float16), i(2, 3), i(2)),
        lambda: bsa.cache_append(q, q, f(3, 2, 16, 64), f(3, 2, 16, 64), i(2, 3), i(2)),
        lambda: bsa.cache_keep(f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2), i(3, 4), i(2), 4),
        lambda: bsa.cache_keep(f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2), i(2, 4), None, 4),
        lambda: bsa.cache_keep(f(3, 4, 16, 64), f(3, 4, 16, 64), i(2, 3), i(2), i(2, 4), i(2), 0),
        lambda: bsa.rotary_nd(q, None, i(8, 2), f(32, dt=torch.float32), (32,)),               # two axes of positions, one of pairs
        lambda: bsa.rotary_nd(q, None, i(8, 1), f(33, dt=torch.float32), (33,)),               # too many pairs
        lambda: bsa.rotary_nd(q, None, i(8, 1), f(31, dt=torch.float32), (32,)),
        lambda: bsa.rotary_nd(q, f(2, 4, 9, 64), i(8, 1), f(32, dt=torch.float32), (32,)),
        lambda: bsa.rotary_nd(q, q, i(8, 1), f(32, dt=torch.float32), (32,), q_out=q, k_out=q),  # rotated twice
        lambda: bsa.rotary_nd(q[:, :, 1:], None, i(7, 1), f(32, dt=torch.float32), (32,), q_out=q[:, :, :-1]),  # shifted overlap
        lambda: bsa.rotary_nd(q, f(2, 4, 8, 64), i(8, 1), f(32, dt=torch.float32), (32,), k_out=q),
    ]
    for n, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            raise RuntimeError(f"call {n} was not refused")


def test_c_entry_points_refuse_bad_arguments():
    from block_sparse_attention import _cabi
    lib = _cabi.load()

    def fwd(**kw):
        a = _cabi.WindowFwdArgs()
        for n in ("q", "k", "v", "out", "status"):
            setattr(a, n, 1 << 20)
        a.B, a.Hq, a.Hkv, a.Sq, a.Sk, a.D = 1, 2, 2, 8, 8, 64
        a.window, a.softmax_scale = 4, 1.0
        for s in ("q_stride", "k_stride", "v_stride", "o_stride"):
            setattr(a, s, (ctypes.c_int64 * 3)(1024, 512, 64))
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.bsa_window_fwd(a, None)

    for kw in (dict(dtype=1), dict(D=80), dict(B=0), dict(Hq=3), dict(q=None), dict(window=0), dict(sinks=129), dict(sinks=-1),
               dict(stream_ctas=-1), dict(stream_ctas=2), dict(team=9), dict(team=-1), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(Sk=0),
               dict(Sk=(1 << 29) + 1), dict(out=(1 << 20) + 2), dict(o_stride=(ctypes.c_int64 * 3)(1024, 512, 60)),
               dict(tree_mask=1 << 20), dict(page_table=1 << 20), dict(page_table=1 << 20, page_size=24, max_pages=1, num_pages=1),
               dict(page_table=1 << 20, page_size=16, max_pages=1, num_pages=1),  # no lengths
               dict(page_table=1 << 20, page_size=16, max_pages=1 << 26, num_pages=1, kv_lens=1 << 20)):
        assert fwd(**kw) < 0, kw
    b = _cabi.WindowBwdArgs()
    assert lib.bsa_window_bwd(b, None) < 0
    for n in ("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv", "workspace", "status"):
        setattr(b, n, 1 << 20)
    b.B, b.Hq, b.Hkv, b.Sq, b.Sk, b.D, b.window, b.softmax_scale = 1, 2, 2, 8, 8, 64, 4, 1.0
    assert lib.bsa_window_bwd(b, None) == -4  # no workspace
    assert lib.bsa_window_bwd_workspace_bytes(1, 2, 2, 8, 8, 64, 4, 4) == 2 * 2 * 128 * 4
    assert lib.bsa_window_bwd_workspace_bytes(1, 2, 2, 8, 8, 64, 0, 4) == 0
    # sinks that later query tiles see keep fp32 sums in the workspace
    assert lib.bsa_window_bwd_workspace_bytes(1, 2, 2, 4096, 4096, 64, 4, 4) > 2 * 2 * 4096 * 4
    r = _cabi.RotaryArgs()
    assert lib.bsa_rotary_nd(r, None) < 0
    st = (ctypes.c_int64 * 3)(1024, 512, 64)
    assert lib.bsa_tree_mask(1 << 20, 1, 65, 1 << 20, None) < 0

    def cache(entry, **kw):
        a = _cabi.CacheArgs(*[1 << 20] * 9, st, st, st, st, 1, 1, 1, 64, 1, 16, 1, 1)
        a.v_cache = 1 << 21
        for n, v in kw.items():
            setattr(a, n, v)
        return entry(a, None)

    for kw in (dict(k_cache=(1 << 20) + 2), dict(k_cache=None), dict(lens=None), dict(page_table=None), dict(v_cache=1 << 20), dict(D=63),
               dict(D=0), dict(B=0), dict(T=0), dict(num_pages=0), dict(page_size=1 << 15, max_pages=1 << 15),
               dict(kc_stride=(ctypes.c_int64 * 3)(1024, 512, 60))):
        assert cache(lib.bsa_cache_append, **kw) < 0 and cache(lib.bsa_cache_keep, **kw) < 0, kw
    for kw in (dict(k=None), dict(v=(1 << 20) + 8), dict(k_stride=(ctypes.c_int64 * 3)(1024, 512, 60))):
        assert cache(lib.bsa_cache_append, **kw) < 0, kw
    for kw in (dict(path=None), dict(path_lens=None), dict(new_lens=None), dict(path_cap=0)):
        assert cache(lib.bsa_cache_keep, **kw) < 0, kw


def test_rule_of_dealing_the_work():
    from block_sparse_attention.window_attn import _deal_work
    whole = (0, 1)
    for items, key_tiles, rows, ragged, want in [
            (296, 100, 128, False, whole),         # a query tile for both places of every SM
            (304, 100, 128, False, (296, 1)),      # a second round for eight of them
            (512, 33, 128, False, whole),          # 66 key tiles at the busiest place, 57 on average
            (148, 100, 128, False, (0, 2)), (148, 7, 4, False, whole),
            (8, 2, 4, False, whole), (8, 4, 4, False, (0, 4)), (8, 33, 4, False, (0, 8)), (8, 300, 4, False, (296, 1)),
            (8, 64, 128, False, (0, 8)), (8, 256, 128, False, (296, 1)),
            (1, 1, 1, True, whole), (1, 7, 128, True, (0, 7)),  # no larger team than there are key tiles
            (1024, 32, 4, True, (296, 1)), (2048, 16, 4, True, whole), (1024, 9, 128, True, whole),
            (0, 5, 1, False, whole), (1 << 20, 1 << 12, 128, False, whole)]:
        assert _deal_work(items, key_tiles, rows, ragged, 148) == want, (items, key_tiles, rows, ragged)


def test_gradient_formula_against_differences():
    g = torch.Generator().manual_seed(0)
    q, do = (torch.randn(1, 2, 9, 4, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(1, 1, 12, 4, generator=g, dtype=torch.float64) for _ in range(2))
    mask = visible(9, 12, 4, 2, 11)[None]
    (dq, dk, dv), _ = gradients(q, k, v, do, mask, 0.5, torch.bfloat16)

    def loss(q, k, v):
        return (attend(q, k, v, mask, 0.5, torch.bfloat16)[0] * do).sum().item()

    h = 1e-5
    for x, dx, at in ((q, dq, 0), (k, dk, 1), (v, dv, 2)):
        for _ in range(12):
            d = torch.randn(x.shape, generator=g, dtype=torch.float64)
            args = [q, k, v]
            args[at] = x + h * d
            up = loss(*args)
            args[at] = x - h * d
            # central differences: h^2 of the third derivative (values of order 10) and 1e-16 / h of rounding
            assert abs((up - loss(*args)) / (2 * h) - (dx * d).sum().item()) < 1e-7
