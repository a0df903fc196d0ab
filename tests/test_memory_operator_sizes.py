"""CPU: sizes that 32 bits do not hold are refused, not passed on by their low 32 bits (2^32 + 4 maps would be normalised as four)."""
import pytest
import torch

BIG = 2 ** 32 + 4


def test_sizes_beyond_32_bits_are_refused():
    from combo_avs_amd.ops.cross_attention import cross_attention
    from combo_avs_amd.ops.groupnorm import group_norm_act
    from combo_avs_amd.ops.rotary import rotary_axes

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")  # (no memory)
    k = meta(1, 3, 1, 8)
    for call in (lambda: group_norm_act(meta(BIG, 1, 1, 1), 1), lambda: group_norm_act(meta(BIG, 8, 1, 1, 1), 2, activation="silu"),
                 lambda: rotary_axes(meta(BIG, 1, 1, 2), meta(1, 1, dtype=torch.float32), (1,)),
                 lambda: rotary_axes(meta(1, BIG, 1, 2), meta(BIG, 1, dtype=torch.float32), (1,)),
                 lambda: rotary_axes(meta(1, 1, BIG, 2), meta(1, 1, dtype=torch.float32), (1,)),
                 lambda: cross_attention(meta(1, BIG, 1, 8), k, k), lambda: cross_attention(meta(1, 1, BIG, 8), k, k),
                 lambda: cross_attention(meta(BIG, 1, 1, 8), meta(BIG, 1, 1, 8), meta(BIG, 1, 1, 8)),
                 lambda: cross_attention(meta(1, 1, 1, 8), meta(1, BIG, 1, 8), meta(1, BIG, 1, 8))):
        with pytest.raises(ValueError):
            call()
