"""Gradients of cross attention in fp16 for upstream gradients of any size, and in bf16 beside it: fp16 holds 30 binades, and a score gradient
p (dp - delta) carries the size of a probability (1 / keys) times that of the upstream gradient, so it has to be held at a scale of its own.

Bounds, in root mean squares against the error of rounding the exact result: a result carries its own rounding and that of p or ds, independent and as
large: sqrt(2), and an eighth more for mantissas that are not spread alike.  Where few states carry a row (values that grow along the states, single
large probabilities) delta = o . do brings the rounding of o as a third: sqrt(3).  The rounding of the exact result includes that of results under
2^-14, where fp16 is coarser; the results themselves may be as small as that, what they are formed from may not lose more than they do."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TWO, THREE = 1.125 * 2 ** 0.5, 1.125 * 3 ** 0.5


def exact(q, k, v, dout, shut=None):
    """-> out, dq, dk, dv [B, L, H, D] in 64 bits on the CPU"""
    q, k, v, g = (t.detach().double().cpu().transpose(1, 2) for t in (q, k, v, dout))
    scale = q.shape[3] ** -0.5
    s = scale * (q @ k.transpose(2, 3))
    if shut is not None:
        s = s.masked_fill(shut, float("-inf"))
    p = torch.softmax(s, -1)
    o = p @ v
    ds = p * (g @ v.transpose(2, 3) - (g * o).sum(-1, keepdim=True))
    return [t.transpose(1, 2) for t in (o, scale * ds @ k, scale * ds.transpose(2, 3) @ q, p.transpose(2, 3) @ g)]


def ours(q, k, v, dout, blocked=None):
    from combo_avs_amd.ops.cross_attention import cross_attention
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, blocked=None if blocked is None else blocked.cuda())
    return [out.detach().cpu()] + [t.cpu() for t in torch.autograd.grad(out, leaves, dout.cuda())]


def ratio(got, want):
    off, own = (got.double() - want).norm(), (want.to(got.dtype).double() - want).norm()
    return float(off / own)


def made(shape, dtype, seed):
    B, H, Lq, Lk, D = shape
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(B, L, H, D, generator=gen) for L in (Lq, Lk, Lk, Lq)]


# (B, H, Lq, Lk, D): blocks of 128 rows and of 32, head dimensions of every tile, keys at hand and long walks, split keys, split rows
SHAPES = [(1, 1, 512, 4096, 64), (1, 1, 300, 16384, 64), (1, 2, 4, 16384, 128), (1, 1, 4096, 512, 128), (1, 2, 2048, 2048, 32), (8, 8, 512, 160, 40), (2, 2, 20, 40, 64)]


@pytest.mark.parametrize("size", [7, 0, -7, -10, -14])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_size_of_the_upstream_gradient(shape, size):
    q, k, v, dout = (t.half() for t in made(shape, torch.float16, shape[3] + shape[4]))
    dout = dout * 2.0 ** size  # (exact, and down to the smallest values of the type)
    for name, a, b in zip(("out", "dq", "dk", "dv"), ours(q, k, v, dout), exact(q, k, v, dout)):
        assert ratio(a, b) <= TWO, (name, ratio(a, b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Lq,Lk,D", [(512, 2048, 64), (512, 512, 128), (24, 1024, 64), (1024, 2048, 32)])
def test_rows_and_states_of_different_gradient_sizes(Lq, Lk, D, dtype):
    """four classes of rows, each with states of its own (a block mask) and upstream gradients of 2^0, 2^-6, 2^-12 and 2^5: every class keeps its digits"""
    q, k, v, dout = made((1, 2, Lq, Lk, D), dtype, 5)
    sizes = torch.tensor([0, -6, -12, 5])
    dout = dout * torch.exp2(sizes[torch.arange(Lq) % 4].float()).view(1, Lq, 1, 1)
    q, k, v, dout = (t.to(dtype) for t in (q, k, v, dout))
    shut = (torch.arange(Lq)[:, None] % 4 != torch.arange(Lk) % 4)[None, None]
    got, want = ours(q, k, v, dout, shut), exact(q, k, v, dout, shut)
    for c in range(4):
        for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
            assert ratio(a[:, c::4], b[:, c::4]) <= THREE, (name, c, ratio(a[:, c::4], b[:, c::4]))


@pytest.mark.parametrize("Lq,Lk,D", [(300, 2048, 64), (512, 1024, 128), (8, 4096, 64), (600, 700, 24)])
def test_score_gradients_that_grow_along_the_walk(Lq, Lk, D):
    """values grow by 2^20 along the states, upstream gradients by 2^16 along the rows, and the first states are seen by nobody: what a walk meets first
    says nothing of what follows"""
    q, k, v, dout = made((1, 2, Lq, Lk, D), torch.float16, 6)
    v = v * torch.exp2(20 * torch.arange(Lk) / Lk - 14).view(1, Lk, 1, 1)
    dout = dout * torch.exp2(16 * torch.arange(Lq) / Lq - 10).view(1, Lq, 1, 1)
    q, k, v, dout = (t.half() for t in (q, k, v, dout))
    shut = (torch.arange(Lk) < 140).expand(1, 1, Lq, Lk).clone()
    got, want = ours(q, k, v, dout, shut), exact(q, k, v, dout, shut)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert ratio(a, b) <= THREE, (name, ratio(a, b))


@pytest.mark.parametrize("Lq,Lk,D", [(300, 20, 64), (4, 300, 128), (260, 600, 32)])
def test_score_gradients_beyond_the_type(Lq, Lk, D):
    """ds past 65504 (dp of 2^25), results that fp16 holds"""
    q, k, v, dout = made((1, 2, Lq, Lk, D), torch.float16, 7)
    q, k, v, dout = (t.half() for t in (q * 2.0 ** -10, k * 2.0 ** -10, v * 2.0 ** 10, dout * 2.0 ** 13))
    got, want = ours(q, k, v, dout), exact(q, k, v, dout)
    assert max(float(t.abs().max()) for t in want) < 65504
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert ratio(a, b) <= THREE, (name, ratio(a, b))
