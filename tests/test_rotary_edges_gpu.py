"""GPU: rotary positions at the edges of what the call takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_k_without_heads():
    from block_sparse_attention import rotary_frequencies, rotary_nd
    q = torch.randn(2, 3, 5, 64, device="cuda").bfloat16()
    pos, freq = torch.arange(5, dtype=torch.int32, device="cuda")[:, None], rotary_frequencies((32,)).cuda()
    want, _ = rotary_nd(q, None, pos, freq, (32,))
    for k in (q[:, :0], torch.empty_strided((2, 0, 5, 64), (0, 320, 1, 5), dtype=q.dtype, device="cuda"), q.new_empty(2, 64, 5, 0).transpose(1, 3)):
        assert k.shape == (2, 0, 5, 64)
        got, none = rotary_nd(q, k, pos, freq, (32,))
        assert torch.equal(got, want) and none.shape == k.shape


def test_slices_of_a_fused_projection_one_of_them_in_place():
    from block_sparse_attention import rotary_frequencies, rotary_nd
    fused = torch.randn(2, 30, 6, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    pos, freq = torch.arange(30, dtype=torch.int32, device="cuda")[:, None], rotary_frequencies((32,)).cuda()
    q, k = fused[:, :, :3], fused[:, :, 3:5]
    want = rotary_nd(q, k, pos, freq, (32,), layout="bshd")
    before = fused.clone()
    a, b = rotary_nd(q, k, pos, freq, (32,), layout="bshd", q_out=q)
    assert a is q and torch.equal(q, want[0]) and torch.equal(b, want[1]) and torch.equal(fused[:, :, 3:], before[:, :, 3:])
    fused.copy_(before)
    rotary_nd(q, None, pos, freq, (32,), layout="bshd", q_out=fused[:, :, 3:])
    assert torch.equal(fused[:, :, 3:], want[0]) and torch.equal(q, before[:, :, :3])
