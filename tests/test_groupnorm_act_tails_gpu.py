"""The activations behind the group norm, value by value and relative to their own size, far into their tails: with a weight of zero the norm's result is
its bias, so a channel's output is act(bias) and, with an upstream gradient of one, the bias' gradient is act'(bias).

Bounds, derived (u = 2^-24).  fp32: GELU by a fitted tail (7e-8 = 1.2 u, its argument 2 u, its evaluation 4 u, the exponential and its exponent 3 u, the
products 3 u) under 16 u of the result, SiLU by an exponential, a sum, a quotient and a product under 8 u; a slope's terms are as large as cdf + |z| density and
sigmoid (1 + |z|), 16 u of these.  16-bit maps round the result (half a step, fp16 2^-25 at least); before that GELU's tail is off by 5e-6 and its
exponent z^2 / 2, rounded twice, by 5e-6 at |z| = 9, SiLU's exponent by |z| u: 2^-16 holds both.  The slopes come back in fp32."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def normal(z):
    return 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("name,reach", [("gelu", 9.0), ("silu", 20.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [4096, 15])
def test_activations_relative_to_their_own_size(name, reach, dtype, width):
    from combo_avs_amd.ops.groupnorm import group_norm_act
    zs = torch.linspace(-reach, reach, 4096 // width * width).view(-1, width).cuda()
    full = dtype == torch.float32
    for bias in zs[::max(1, len(zs) // 16)]:
        b = bias.clone().requires_grad_(True)
        x = torch.randn(1, width, 1, 1, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        y = group_norm_act(x, 1, torch.zeros(width, device="cuda"), b, activation=name)
        (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
        z = bias.double().cpu()
        if name == "gelu":
            c, d = normal(z)
            want, slope, size = z * c, c + z * d, c + z.abs() * d
        else:
            c = torch.sigmoid(z)
            want, slope, size = z * c, c * (1 + z * (1 - c)), c * (1 + z.abs())
        off = (y.detach().double().cpu().view(-1) - want).abs()
        rel = (16 if name == "gelu" else 8) * U if full else torch.finfo(dtype).eps / 2 + 2.0 ** -16
        tol = rel * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
        assert (off <= tol).all(), (float((off / tol).max()), float(z[(off / tol).argmax()]))
        off = (db.double().cpu() - slope).abs()
        tol = (16 * U if full else 2.0 ** -16) * size + 1e-37
        assert (off <= tol).all(), (float((off / tol).max()), float(z[(off / tol).argmax()]))
