"""What goes past autograd's backward pass: forward-mode tangents are refused (the ops have none) and never dropped, traces hold the call."""
import warnings

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def calls(seed):
    """name -> (call of its first tensor, that tensor, the other tensors that may carry a tangent)"""
    from combo_avs_amd.ops.cross_attention import cross_attention
    from combo_avs_amd.ops.groupnorm import group_norm_act
    from combo_avs_amd.ops.rotary import rotary_axes
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen)
    m, w, b = rand(2, 8, 6, 6).cuda().contiguous(memory_format=torch.channels_last), rand(8).cuda(), rand(8).cuda()
    x, pos = rand(2, 40, 4, 16).cuda(), rand(40, 1).cuda()
    q, k, v = (rand(2, n, 4, 16).bfloat16().cuda() for n in (40, 70, 70))
    lengths, blocked = torch.tensor([70, 30]).cuda(), (rand(2, 1, 40, 70) > 1).cuda()
    return {"norm": (lambda m, w=w, b=b: group_norm_act(m, 2, w, b, activation="silu"), m, (w, b)),
            "rotary": (lambda x, pos=pos: rotary_axes(x, pos, (4,)), x, (pos,)),
            "cross": (lambda q, k=k, v=v: cross_attention(q, k, v, lengths, blocked), q, (k, v))}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["norm", "rotary", "cross"])
def test_tangents_are_not_dropped(name, grad):
    call, first, rest = calls(1)[name]
    with torch.set_grad_enabled(grad):
        want = call(first)
        for i in range(1 + len(rest)):
            with forward_ad.dual_level():
                args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate((first, *rest))]
                with pytest.raises(NotImplementedError, match="jvp"):
                    call(*args)
                assert torch.equal(call(first), want)  # (no tangent: as outside)
        assert torch.equal(call(first), want)


@pytest.mark.parametrize("name", ["norm", "rotary", "cross"])
def test_traces_hold_the_call(name):
    call, first, _ = calls(2)[name]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # (sizes are checked in Python)
        traced = torch.jit.trace(call, (first,))
    for seed in (3, 4):
        other = calls(seed)[name][1]
        spoil = [torch.full_like(other, float("nan")) for _ in range(4)]  # memory that an output without its launch would show
        del spoil
        assert torch.equal(traced(other), call(other))
