"""CPU: plans and checks of the positional, windowed and cached operators at their edges."""
import time
from types import SimpleNamespace

import pytest
import torch


def meta(shape, strides, dtype=torch.bfloat16):
    """What the checks look at: a tensor on a GPU."""
    return torch.Size(shape), tuple(strides), dtype, torch.device("cuda", 0), True


def test_rotation_of_a_k_without_heads():
    from block_sparse_attention.rotary import _rotary_plan
    q, pos, freq = meta((2, 3, 5, 64), (960, 320, 64, 1)), meta((5, 1), (1, 1), torch.int32), meta((32,), (1,), torch.float32)
    for strides in ((0, 320, 64, 1), (0, 1, 5, 15)):  # (contiguous() gives an empty tensor back as it is)
        plan = _rotary_plan(q, meta((2, 0, 5, 64), strides), pos, freq, (32,), True, False, None, None, "bhsd")
        assert plan.direct and not plan.empty and plan.k_shape == (2, 0, 5, 64)


def elements(shape, strides, size, at):
    """Addresses of every byte."""
    places = torch.tensor([at])
    for n, s in zip(shape, strides):
        places = (places[:, None] + torch.arange(n) * s * size).flatten()
    return set((places[:, None] + torch.arange(size)).flatten().tolist())


def test_views_meet_exactly_where_they_share_a_byte():
    from block_sparse_attention.overlap import _meet, span_bytes, spread
    g = torch.Generator().manual_seed(0)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    met = 0
    for n in range(4000):
        views = []
        for _ in range(2):
            shape = [pick(1, 5) for _ in range(pick(1, 5))]
            if n % 2:  # slices of a fused tensor, dimensions in any order
                inner, strides = 1, []
                for m in reversed(shape):
                    strides.insert(0, inner)
                    inner *= m + pick(0, 3)
                order = torch.randperm(len(shape), generator=g).tolist()
                shape, strides = [shape[i] for i in order], [strides[i] for i in order]
            else:
                strides = [pick(0, 12) for _ in shape]
            views.append((tuple(shape), tuple(strides), (1, 2, 4)[pick(0, 3)]))
        a, b = views
        distance = pick(-span_bytes(*b) - 2, span_bytes(*a) + 2)
        shared = elements(*a, 0) & elements(*b, distance)
        assert _meet(a, b, distance) == bool(shared), (a, b, distance)
        met += bool(shared)
        own = elements(a[0], a[1], 1, 0)
        if spread(*a[:2]):  # (strides that do not nest are refused also where they happen to miss each other)
            assert len(own) == torch.Size(a[0]).numel()
        if n % 2:
            assert spread(*a[:2])
    assert 1000 < met < 3500


def test_large_views_are_compared_quickly():
    from block_sparse_attention.overlap import _meet
    tokens, heads, D = 1 << 20, 48, 128
    rows = (1, tokens, 16, D), (tokens * heads * D, heads * D, D, 1), 2
    t0 = time.time()
    for other in range(1, 3):  # q, k, v of one projection
        assert not _meet(rows, rows, other * 16 * D * 2)
    assert _meet(rows, rows, 16 * D * 2 - 2)  # k begins in q's last channel
    assert _meet(rows, rows, 2 * 16 * D * 2 + 2)  # v ends in the next token's first
    page = (1 << 17, 8, 64, D), (2 * 8 * 64 * D, 64 * D, D, 1), 2
    assert not _meet(page, page, 8 * 64 * D * 2) and _meet(page, page, 8 * 64 * D * 2 - 2)
    across = (1, 16, tokens, D), (tokens * heads * D, tokens * D, D, 1), 2  # another order of the same memory
    assert _meet(rows, across, 64)
    assert time.time() - t0 < 1


class _FakeCuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: reaches the checks behind the device check."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    is_cuda = property(lambda self: True)


def test_outputs_that_share_memory_are_refused(monkeypatch):
    import block_sparse_attention as bsa
    from block_sparse_attention import _cabi
    monkeypatch.setattr(_cabi, "load", lambda: SimpleNamespace(bsa_num_sms=lambda device: 148, bsa_window_bwd_workspace_bytes=lambda *sizes: 16))
    f = lambda *s, dt=torch.bfloat16: _FakeCuda(torch.zeros(*s, dtype=dt))  # noqa: E731
    i = lambda *s: _FakeCuda(torch.zeros(*s, dtype=torch.int32))  # noqa: E731
    new = lambda: f(2, 2, 8, 64)  # noqa: E731
    lse, wide = f(2, 2, 8, dt=torch.float32), f(2, 2, 16, 64)
    a, b = wide[:, :, :8], wide[:, :, 4:12]  # eight rows each, four of them in common
    odd = f(2 * 2 * 8 * 64 + 1)[1:].view(2, 2, 8, 64)  # not 16-byte aligned
    bwd = lambda q=new(), k=new(), v=new(), do=new(), **kw: bsa.window_attn_bwd(do, q, k, v, new(), lse, 4, **kw)  # noqa: E731
    pool, table, n = f(6, 2, 16, 64), i(2, 3), i(2)
    pos, freq = i(8, 1), f(32, dt=torch.float32)
    calls = [
        lambda: bsa.window_attn_fwd(new(), a, new(), 4, out=b),
        lambda: bsa.window_attn_fwd(new(), new(), a, 4, out=b),
        lambda: bsa.window_attn_fwd(a, new(), new(), 4, out=b),                    # q itself, but shifted
        lambda: bsa.window_attn_fwd(a, a, new(), 4, out=a),
        lambda: bsa.window_attn_fwd(new(), odd, new(), 4, out=odd),
        lambda: bsa.window_attn_fwd(a, new(), new(), 4, lse=wide.view(torch.float32).view(-1)[7:263].as_strided((2, 2, 8), (16, 8, 1))),
        lambda: bsa.window_attn_fwd(new(), new(), new(), 4, out=new()[:, :1].expand(2, 2, 8, 64)),
        lambda: bsa.window_attn_fwd(new(), new(), new(), 4, out=wide.as_strided((2, 2, 8, 64), (2048, 1024, 8, 1))),
        lambda: bsa.window_attn_fwd(new(), new(), new(), 4, lse=lse[:, :1].expand(2, 2, 8)),
        lambda: bwd(dk=a, dv=b),
        lambda: bwd(dk=odd, dv=odd),
        lambda: bwd(dq=odd, dv=odd),
        lambda: bwd(q=a, dq=a),
        lambda: bwd(do=a, dq=b),
        lambda: bwd(v=a, dk=b),
        lambda: bwd(dk=wide.as_strided((2, 2, 8, 64), (2048, 1024, 32, 1))),
        lambda: bsa.cached_attn_fwd(pool[:2, :, :8], pool, f(6, 2, 16, 64), table, n, out=pool[2:4, :, :8]),
        lambda: bsa.cached_attn_fwd(new(), pool, pool, i(2, 3), n, out=pool[:2, :, 8:]),
        lambda: bsa.cached_attn_fwd(a, pool, pool, table, n, out=b),
        lambda: bsa.cache_append(new(), new(), pool[:4], pool[1:5], table, n),
        lambda: bsa.cache_append(pool[:2, :, :8], new(), pool, f(6, 2, 16, 64), table, n),
        lambda: bsa.cache_append(new(), pool[3:5, :, 2:10], f(6, 2, 16, 64), pool, table, n),
        lambda: bsa.cache_append(new(), new(), wide.as_strided((3, 2, 16, 64), (512, 256, 16, 1)), f(3, 2, 16, 64), table, n),
        lambda: bsa.cache_keep(pool[:4], pool[1:5], table, n, i(2, 4), n, 4),
        lambda: bsa.rotary_nd(a, None, pos, freq, (32,), q_out=b),
        lambda: bsa.rotary_nd(a, b, pos, freq, (32,), q_out=a, k_out=b),             # both in place, but four rows are common
        lambda: bsa.rotary_nd(a, b, pos, freq, (32,), q_out=a),
        lambda: bsa.rotary_nd(new(), new(), pos, freq, (32,), q_out=a, k_out=a),
        lambda: bsa.rotary_nd(a, f(2, 0, 8, 64), pos, freq, (32,), q_out=b),         # the other one empty
    ]
    for at, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            raise RuntimeError(f"call {at} was not refused")


def test_every_operator_struct_matches_the_header():
    """Names, types and array lengths of the header's fields, in order."""
    import ctypes
    import os
    import re
    from block_sparse_attention import _cabi
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "bsa_b200.h")).read()
    plain = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
    for struct, cls in (("bsa_window_fwd_args", _cabi.WindowFwdArgs), ("bsa_window_bwd_args", _cabi.WindowBwdArgs),
                        ("bsa_rotary_args", _cabi.RotaryArgs), ("bsa_cache_args", _cabi.CacheArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, flags=re.S).group(1)
        fields = []
        for decl in filter(None, (d.strip() for d in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"))):
            kind, names = re.match(r"(?:const\s+)?(\w+)\s*(.*)", decl, flags=re.S).groups()
            for name in names.split(","):
                star, name, count = re.match(r"\s*(\*?)\s*(\w+)(?:\[(\d+)\])?\s*$", name).groups()
                one = ctypes.c_void_p if star else plain[kind]
                fields.append((name, one * int(count) if count else one))
        assert [f[0] for f in fields] == [f[0] for f in cls._fields_], struct
        for (name, want), (_, got) in zip(fields, cls._fields_):
            assert (got is want) or (issubclass(got, ctypes.Array) and got._type_ is want._type_ and got._length_ == want._length_), (struct, name)
