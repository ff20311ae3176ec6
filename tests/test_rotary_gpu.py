"""GPU parity of rotary positions with several axes against the definition in 64 bits."""
import pytest
import torch

from plain_ops import assert_within, half_step, rotate

pytestmark = pytest.mark.gpu

# dtype, B, Hq, Hk, S, D, pairs, interleaved
CASES = [
    (torch.bfloat16, 1, 1, 1, 1, 128, (64,), True),
    (torch.bfloat16, 2, 5, 2, 77, 128, (22, 21, 21), True),
    (torch.bfloat16, 2, 3, 1, 33, 128, (16, 24, 24), False),
    (torch.float16, 3, 2, 2, 50, 96, (16, 16), False),       # part of the head
    (torch.float16, 1, 4, 4, 41, 64, (3, 5, 2, 1), True),    # four axes, a chunk half turned
    (torch.float16, 1, 2, 1, 20, 72, (18, 18), False),       # halves that 16-byte chunks do not fit
    (torch.float32, 2, 2, 2, 65, 64, (0, 32), True),         # an axis without pairs
    (torch.float32, 1, 3, 1, 19, 20, (4, 4), False),
    (torch.float32, 1, 1, 1, 9, 6, (1, 2), True),
    (torch.bfloat16, 1, 2, 2, 9, 512, (100, 100, 56), False),
]


def tolerance(ref, size, dtype):
    # sine and cosine to 2^-22, two 32-bit products and a sum, then the rounding to dtype
    u = half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return u * ref.abs() + 2.0 ** -21 * size * (1 + u) + tiny


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotation(case, layout, inverse):
    from block_sparse_attention import rotary_frequencies, rotary_nd
    dtype, B, Hq, Hk, S, D, pairs, interleaved = case
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(B, h, S, D, generator=g).to(dtype) for h in (Hq, Hk))
    pos = torch.randint(-100000, 1000000, (B, S, len(pairs)), generator=g, dtype=torch.int32)
    pos[0, 0] = 0
    freq = rotary_frequencies(pairs)
    put = (lambda t: t) if layout == "bhsd" else (lambda t: t.transpose(1, 2).contiguous())
    a, b = rotary_nd(put(q).cuda(), put(k).cuda(), pos.cuda(), freq.cuda(), pairs, interleaved=interleaved, inverse=inverse, layout=layout)
    for got, x in ((a, q), (b, k)):
        got = got if layout == "bhsd" else got.transpose(1, 2)
        ref, size = rotate(x.double(), pos, freq, pairs, interleaved, inverse)
        assert_within(got, ref, tolerance(ref, size, dtype), "rotated")
        assert torch.equal(got[..., 2 * sum(pairs):].cpu(), x[..., 2 * sum(pairs):])


def test_far_positions_keep_their_angle():
    from block_sparse_attention import rotary_nd
    pos = torch.tensor([[2 ** 31 - 1], [-2 ** 31], [1 << 24], [12345678]], dtype=torch.int32)
    x = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(0))
    freq = torch.rand(32, generator=torch.Generator().manual_seed(1)) + 0.5
    got, none = rotary_nd(x.cuda(), None, pos.cuda(), freq.cuda(), (32,))
    ref, size = rotate(x.double(), pos[None], freq, (32,), True)
    assert none is None
    assert_within(got, ref, tolerance(ref, size, torch.float32), "rotated")


def test_views_in_place_and_gradient():
    from block_sparse_attention import rotary_embedding, rotary_frequencies, rotary_nd
    g = torch.Generator().manual_seed(2)
    pairs = (12, 20)
    freq = rotary_frequencies(pairs, theta=500.0, shared_ladder=True).cuda()
    fused = torch.randn(2, 30, 6, 64, generator=g).bfloat16().cuda()  # tokens, then q heads, k heads, v heads
    pos = torch.randint(0, 99, (30, 2), generator=g, dtype=torch.int32).cuda()
    want = rotary_nd(fused[:, :, :3].contiguous(), fused[:, :, 3:4].contiguous(), pos, freq, pairs, layout="bshd")
    v = fused[:, :, 4:].clone()
    q, k = fused[:, :, :3], fused[:, :, 3:4]
    got = rotary_nd(q, k, pos, freq, pairs, layout="bshd", q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, :, 4:], v)
    # unaligned rows take the element form
    odd = torch.randn(2, 3, 30, 67, generator=g).bfloat16().cuda()[..., 3:]
    a, _ = rotary_nd(odd, None, pos, freq, pairs)
    b, _ = rotary_nd(odd.contiguous(), None, pos, freq, pairs)
    assert torch.equal(a, b)
    # the gradient: rotation back, q used twice, k broadcast over heads
    x = torch.randn(2, 4, 30, 64, generator=g).cuda().requires_grad_()
    y = torch.randn(2, 1, 30, 64, generator=g).cuda().requires_grad_()
    wq, wk = (torch.randn(2, 4, 30, 64, generator=g).cuda() for _ in range(2))
    rq, rk = rotary_embedding(x, y.expand(2, 4, 30, 64), pos, freq, pairs, interleaved=False)
    ((rq * wq).sum() + (rk * wk).sum()).backward()
    p3 = pos.cpu()[None].expand(2, 30, 2)
    ref, size = rotate(wq.double().cpu(), p3, freq.cpu(), pairs, False, True)
    assert_within(x.grad, ref, tolerance(ref, size, torch.float32), "dq")
    ref, size = rotate(wk.double().cpu(), p3, freq.cpu(), pairs, False, True)
    ref, size = ref.sum(1, keepdim=True), size.sum(1, keepdim=True)
    assert_within(y.grad, ref, tolerance(ref, size, torch.float32) + 4 * 2.0 ** -23 * size, "dk")
    # only one of the two outputs is used
    rq, rk = rotary_embedding(x, y, pos, freq, pairs)
    gy, = torch.autograd.grad(rk.sum(), y)
    assert gy.shape == y.shape
    # differences: <w, R x> is linear in x
    d = torch.randn(x.shape, generator=g).cuda()
    with torch.no_grad():
        up, _ = rotary_nd(x + d, None, pos, freq, pairs, interleaved=False)
        dn, _ = rotary_nd(x - d, None, pos, freq, pairs, interleaved=False)
    diff = ((up.double() - dn.double()) * wq.double()).sum() / 2
    dot = (x.grad.double() * d.double()).sum()
    assert abs((diff - dot).item()) <= 2.0 ** -19 * ((up.abs() + dn.abs()).double() * wq.abs().double()).sum().item()


def test_graph_and_stream():
    from block_sparse_attention import rotary_frequencies, rotary_nd
    freq = rotary_frequencies((32, 32)).cuda()
    q, k = torch.randn(2, 4, 9, 128, device="cuda").half(), torch.randn(2, 2, 9, 128, device="cuda").half()
    pos = torch.randint(0, 1000, (2, 9, 2), dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = rotary_nd(q, k, pos, freq, (32, 32))
    torch.cuda.current_stream().wait_stream(side)
    b = rotary_nd(q, k, pos, freq, (32, 32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = rotary_nd(q, k, pos, freq, (32, 32))
    pos += 5
    graph.replay()
    b = rotary_nd(q, k, pos, freq, (32, 32))
    assert torch.equal(res[0], b[0]) and torch.equal(res[1], b[1])


def test_q_alone_has_a_gradient():
    from block_sparse_attention import rotary_embedding, rotary_frequencies
    freq = rotary_frequencies((32,)).cuda()
    pos = torch.arange(7, dtype=torch.int32, device="cuda")[:, None]
    x = torch.randn(1, 2, 7, 64, device="cuda", requires_grad=True)
    y, none = rotary_embedding(x, None, pos, freq, (32,))
    assert none is None
    (y * y).sum().backward()
    # a rotation keeps lengths: the gradient of the squared norm is 2 x (two rotations' 32-bit roundings)
    torch.testing.assert_close(x.grad, 2 * x.detach(), rtol=0, atol=2.0 ** -18)


def test_every_head_dimension_and_pair_count():
    """Every form's edges: chunks that are turned in part, halves that do not fit chunks, tails."""
    from block_sparse_attention import rotary_frequencies, rotary_nd
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.bfloat16, torch.float32):
        for D in (2, 4, 8, 16, 24, 62, 64, 200, 256):
            for P in sorted({1, D // 2, max(1, D // 4), max(1, D // 2 - 1)}):
                for interleaved in (True, False):
                    x = torch.randn(1, 3, 5, D, generator=g).to(dtype)
                    pos = torch.randint(0, 500, (1, 5, 1), generator=g, dtype=torch.int32)
                    freq = rotary_frequencies((P,))
                    got, _ = rotary_nd(x.cuda(), None, pos.cuda(), freq.cuda(), (P,), interleaved=interleaved)
                    ref, size = rotate(x.double(), pos, freq, (P,), interleaved)
                    assert_within(got, ref, tolerance(ref, size, dtype), f"D {D}, P {P}")
                    assert torch.equal(got[..., 2 * P:].cpu(), x[..., 2 * P:])


@pytest.mark.parametrize("D", [64, 20])  # 16-byte chunks, and rows that they do not fit
@pytest.mark.parametrize("interleaved", [True, False])
def test_bad_frequencies_show_in_their_own_pairs(D, interleaved):
    from block_sparse_attention import rotary_nd
    P = D // 2
    x = torch.randn(1, 2, 3, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()
    freq = torch.rand(P, generator=torch.Generator().manual_seed(1))
    freq[1], freq[4] = float("nan"), float("-inf")
    got, _ = rotary_nd(x, None, torch.arange(1, 4, dtype=torch.int32)[:, None].cuda(), freq.cuda(), (P,), interleaved=interleaved)
    bad = torch.zeros(D, dtype=torch.bool)
    for p in (1, 4):
        bad[[2 * p, 2 * p + 1] if interleaved else [p, P + p]] = True
    assert torch.equal(got.isnan().cpu(), bad.expand(1, 2, 3, D))
