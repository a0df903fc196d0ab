"""Group norm with an activation on channels-last maps (csrc/groupnorm_act.hip, ops/groupnorm.group_norm_act) against the formulas in
64 bits.

Tolerances, derived (u = 2^-24): x - mean is off by 16 u (|x| + |mean|) (the tree of the mean, one subtraction), rstd by 64 u (at most 64
values in a thread's shifted sum at these sizes, plus the joins), the activation by 2^-21 (1 + |z|) (exp2 of z log2 e, erf); the slopes stay
under 1.2.  In the gradient every product and mean adds a few u: 32 u of each term's size.  dw, db: a thread adds at most 98 values, the joins
30 more: 128 u of the sum of absolute values.  Then one rounding, half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def phi(z):
    return 0.5 * torch.erfc(-z / math.sqrt(2))


def act(z, name):
    return {"none": z, "relu": z.clamp_min(0), "silu": z * torch.sigmoid(z), "gelu": z * phi(z)}[name]


def slope(z, name):
    s = torch.sigmoid(z)
    return {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s)),
            "gelu": phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[name]


def check(x, dy, G, w, b, name, eps=1e-5):
    """x, dy [B, C, ...] channels last on the GPU; w, b [C]"""
    from combo_avs_amd.ops.groupnorm import group_norm_act
    B, C = x.shape[:2]
    half = torch.finfo(x.dtype).eps / 2
    floor = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    X = x.double().cpu().reshape(B, G, C // G, -1)
    W, Bb = (t.double().cpu().reshape(1, G, -1, 1) for t in (w, b))
    mean = X.mean((2, 3), keepdim=True)
    rstd = (((X - mean) ** 2).mean((2, 3), keepdim=True) + eps).rsqrt()
    xh = (X - mean) * rstd
    z = xh * W + Bb
    dy = torch.where((z.abs() < 1e-3).reshape(dy.shape).to(dy.device), torch.zeros_like(dy), dy)  # a ReLU's slope is not defined by rounding
    dy = dy.contiguous(memory_format=torch.channels_last if dy.dim() == 4 else torch.channels_last_3d)
    xs, ws, bs = x.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = group_norm_act(xs, G, ws, bs, eps, name)
    assert y.shape == x.shape and y.dtype == x.dtype and y.stride() == torch.empty_like(x).stride()
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), dy)
    assert dw.dtype == w.dtype and db.dtype == b.dtype and dx.dtype == x.dtype
    off_z = W.abs() * (16 * U * (X.abs() + mean.abs()) * rstd + 64 * U * xh.abs()) + 2 * U * (z.abs() + Bb.abs())
    want = act(z, name)
    tol = half * want.abs() + 1.2 * off_z + 2.0 ** -21 * (1 + z.abs()) + floor
    off = (y.detach().double().cpu().reshape(X.shape) - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    D = dy.double().cpu().reshape(X.shape)
    dz = D * slope(z, name)
    dxh = dz * W
    want = rstd * (dxh - dxh.mean((2, 3), keepdim=True) - xh * (dxh * xh).mean((2, 3), keepdim=True))
    bend = (0 if name in ("none", "relu") else 1) * off_z + 2.0 ** -21 * (1 + z.abs())  # second derivatives stay under 1
    off_xh = 16 * U * (X.abs() + mean.abs()) * rstd + 64 * U * xh.abs()
    size = (D * W).abs()
    off_dxh = size * bend + 32 * U * size
    tol = half * want.abs() + floor + rstd * (off_dxh + off_dxh.mean((2, 3), keepdim=True) + 32 * U * size.mean((2, 3), keepdim=True)
                                              + off_xh * (dxh * xh).mean((2, 3), keepdim=True).abs()
                                              + xh.abs() * (off_dxh * xh.abs() + size * off_xh + 32 * U * size * xh.abs()).mean((2, 3), keepdim=True))
    off = (dx.double().cpu().reshape(X.shape) - want).abs()
    assert (off <= tol * (1 + 128 * U)).all(), float((off / tol).max())
    half_w = torch.finfo(w.dtype).eps / 2
    for got, terms, more in ((dw, dz * xh, D.abs() * (bend * xh.abs() + 1.2 * off_xh)), (db, dz, D.abs() * bend)):
        want = terms.sum((0, 3)).reshape(C)
        tol = half_w * want.abs() + 128 * U * terms.abs().sum((0, 3)).reshape(C) + more.sum((0, 3)).reshape(C) + 1e-30
        off = (got.double().cpu() - want).abs()
        assert (off <= tol).all(), float((off / tol).max())


def made(shape, dtype, seed, offset=0.0):
    gen = torch.Generator().manual_seed(seed)
    fmt = torch.channels_last if len(shape) == 4 else torch.channels_last_3d
    scale = (torch.rand(shape[1], generator=gen) + 0.5).view(1, -1, *[1] * (len(shape) - 2))
    x = (torch.randn(shape, generator=gen) * scale + torch.randn(shape[1], generator=gen).view(scale.shape) + offset).to(dtype)
    dy = torch.randn(shape, generator=gen).to(dtype)
    w, b = torch.rand(shape[1], generator=gen) + 0.5, torch.randn(shape[1], generator=gen) * 0.5
    return x.cuda().contiguous(memory_format=fmt), dy.cuda().contiguous(memory_format=fmt), w.cuda(), b.cuda()


SHAPES = [  # (B, C, H, W), groups: one channel a group, one group, odd channel counts, one launch and two, more vectors than threads
    ((1, 32, 7, 7), 32), ((2, 60, 9, 13), 6), ((1, 7, 5, 3), 1), ((3, 256, 56, 56), 32), ((2, 96, 2, 2), 8), ((1, 2048, 3, 3), 32),
    ((1, 4096, 2, 2), 1), ((2, 36, 61, 67), 4), ((1, 1, 40, 40), 1), ((2, 24, 3, 5, 7), 3), ((1, 130, 97, 31), 2), ((40, 64, 28, 28), 32),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_matches_the_formulas(shape, groups, dtype):
    names = ["none", "relu", "silu", "gelu"]
    check(*made(shape, dtype, sum(shape))[:2], groups, *made(shape, dtype, sum(shape))[2:], names[(sum(shape) + groups) % 4])


@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_every_activation(name, dtype):
    for shape in ((2, 16, 6, 5), (1, 16, 130, 64)):
        x, dy, w, b = made(shape, dtype, 11)
        check(x, dy, 4, w, b, name)


def test_a_large_offset_keeps_the_variance():
    """offset 3000 with a spread of about 1: the sum of squares in fp32 would keep nothing of the variance"""
    x, dy, w, b = made((1, 16, 20, 20), torch.float32, 1, offset=3000.0)
    check(x, dy, 4, w, b, "none")
    x, dy, w, b = made((1, 16, 200, 200), torch.float32, 2, offset=3000.0)
    check(x, dy, 4, w, b, "silu")


def test_half_parameters_misaligned_maps_no_parameters():
    from combo_avs_amd.ops.groupnorm import group_norm_act
    x, dy, w, b = made((2, 16, 9, 7), torch.bfloat16, 4)
    check(x, dy, 4, w.bfloat16(), b.bfloat16(), "silu")
    flat = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)
    odd = flat[1:].view(2, 9, 7, 16).permute(0, 3, 1, 2)
    odd.copy_(x)
    assert odd.is_contiguous(memory_format=torch.channels_last) and odd.data_ptr() % 4
    check(odd, dy, 4, w, b, "gelu")
    xs = x.clone().requires_grad_(True)
    one, zero = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    a, c = group_norm_act(xs, 4, activation="relu"), group_norm_act(xs, 4, one, zero, activation="relu")
    assert torch.equal(a, c) and torch.equal(torch.autograd.grad(a, xs, dy)[0], torch.autograd.grad(c, xs, dy)[0])
    ws = w.clone().requires_grad_(True)  # (only the weight asks for its gradient; an expanded gradient comes in)
    y = group_norm_act(x, 4, ws, b, activation="none")
    (dw,) = torch.autograd.grad(y.sum(), ws)
    assert dw.shape == (16,) and torch.isfinite(dw).all()


def test_empty_batch():
    from combo_avs_amd.ops.groupnorm import group_norm_act
    x = torch.empty(0, 8, 4, 4, device="cuda").contiguous(memory_format=torch.channels_last).requires_grad_(True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = group_norm_act(x, 2, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == x.shape and dx.shape == x.shape and torch.equal(dw, torch.zeros(8, device="cuda"))


def test_gradient_agrees_with_differences():
    from combo_avs_amd.ops.groupnorm import group_norm_act
    x, d, w, b = made((1, 8, 5, 4), torch.float32, 8)
    for name in ("silu", "gelu"):
        xs = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad((group_norm_act(xs, 2, w, b, activation=name) * d).sum(), xs)
        h = 2.0 ** -6
        diff = ((group_norm_act(x + h * d, 2, w, b, activation=name) - group_norm_act(x - h * d, 2, w, b, activation=name)) * d).double().sum() / (2 * h)
        # truncation h^2 / 6 of a third derivative of order |d|^3 per value (160 values, |d| of order 1): 160 * 8 * 2^-12 / 6 = 0.05;
        # roundings 160 * 2^-22 / 2^-6: 0.003
        assert abs(float((g * d).double().sum() - diff)) < 0.06


def test_runs_repeat_bit_for_bit_on_streams_and_in_graphs():
    from combo_avs_amd.ops.groupnorm import group_norm_act
    for shape in ((2, 64, 9, 9), (2, 64, 80, 80)):
        x, dy, w, b = made(shape, torch.bfloat16, 6)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]

        def step():
            y = group_norm_act(*([leaves[0], 8] + leaves[1:]), activation="silu")
            return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
        eager = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(eager, other))
        graph, twin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        with torch.cuda.graph(twin, pool=graph.pool()):
            held2 = step()
        for seed in range(3):
            with torch.no_grad():
                x.copy_(torch.randn(shape, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(step(), held))
            twin.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(step(), held2))
