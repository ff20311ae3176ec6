"""CPU: plans and checks of the positional, windowed and cached operators at their edges."""
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
