"""The values behind the pairs pass through rotary_axes bit for bit, whatever they are, and the pairs before them do not depend on them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,sections", [(80, (16, 18)), (10, (3,)), (16, (0, 7)), (64, (1,)), (256, (5, 50)), (8, (0,))])
def test_values_behind_the_pairs_pass_through(D, sections, interleaved, dtype):
    from combo_avs_amd.ops.rotary import rotary_axes
    gen = torch.Generator().manual_seed(D)
    pos = torch.rand(9, len(sections), generator=gen).cuda() * 50
    plain = torch.randn(2, 9, 3, D, generator=gen).to(dtype)
    start = 2 * sum(sections)
    odd = plain.clone()
    for i, v in enumerate((float("inf"), -0.0, float("nan"), -float("inf"))):  # next to finite values, on either side of a pair of places
        odd[..., start + i:start + i + 1] = v
    odd[..., start + 5::8] = float("inf")
    for x in (plain, odd):
        g = x.cuda().requires_grad_(True)
        y = rotary_axes(g, pos, sections, interleaved=interleaved)
        (dx,) = torch.autograd.grad(y, g, x.cuda())
        for got in (y.detach(), dx):
            kept, given = got[..., start:].contiguous().cpu(), x[..., start:].contiguous()
            kind = torch.int32 if dtype == torch.float32 else torch.int16
            assert torch.equal(kept.view(kind), given.view(kind))
        if x is plain:
            want = y.detach(), dx
        else:
            assert torch.equal(y.detach()[..., :start], want[0][..., :start]) and torch.equal(dx[..., :start], want[1][..., :start])
