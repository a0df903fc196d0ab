"""Weight and bias gradients are fp32 sums over a map of any type: they are as exact as fp32 sums of the formulas' terms, not as the map's type.

Bound, derived (u = 2^-24), in root mean squares over the channels against the sum of the terms' absolute sizes: what is off in the same direction
everywhere stays - act's fitted tail 1.2 u, its reciprocal and its exponential half an u each -, what is off at random falls with the number of terms: the
sums in at most 150 steps a thread 4 u of a thread's share, of which 200 and more are joined, 0.3 u.  2.5 u."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("name", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,groups", [((3, 60, 117, 93), 6), ((4, 64, 24, 24), 8)])
def test_parameter_gradients_have_the_digits_of_fp32(shape, groups, dtype, name):
    from combo_avs_amd.ops.groupnorm import group_norm_act
    B, C = shape[:2]
    gen = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(shape, generator=gen).to(dtype).cuda().contiguous(memory_format=torch.channels_last) for _ in range(2))
    dy = dy.abs()  # (one sign: what is off in the same direction everywhere does not cancel)
    w, b = (t.cuda().requires_grad_(True) for t in (torch.rand(C, generator=gen) + 0.5, torch.randn(C, generator=gen) * 0.5))
    dw, db = torch.autograd.grad(group_norm_act(x, groups, w, b, activation=name), (w, b), dy)
    X, D = (t.double().cpu().reshape(B, groups, C // groups, -1) for t in (x, dy))
    W, Bb = (t.detach().double().cpu().reshape(1, groups, -1, 1) for t in (w, b))
    xh = (X - X.mean((2, 3), keepdim=True)) * (X.var((2, 3), unbiased=False, keepdim=True) + 1e-5).rsqrt()
    z = xh * W + Bb
    if name == "gelu":
        c, d = 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        slope, size = c + z * d, c + z.abs() * d
    else:
        c = torch.sigmoid(z)
        slope, size = c * (1 + z * (1 - c)), c * (1 + z.abs())
    for got, terms, most in ((dw, D * slope * xh, D * size * xh.abs()), (db, D * slope, D * size)):
        off = got.double().cpu() - terms.sum((0, 3)).reshape(C)
        assert off.norm() <= 2.5 * U * most.sum((0, 3)).norm(), float(off.norm() / (U * most.sum((0, 3)).norm()))
