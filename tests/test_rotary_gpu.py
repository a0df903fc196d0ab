"""Rotary positions over several axes (csrc/rotary.hip, ops/rotary.py) against the definition in 64 bits.

Tolerance, derived: the angle is off by at most 2^-25 of a turn (rounding of the reduced angle to fp32; 2e-7 rad), sincospi by 2 ulp, the
two products and their sum by 3 * 2^-24: together under 6e-7 (|lo| + |hi|); then one rounding to the tensor's type, half a step."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def defined(x, pos, sections, base, interleaved, shared, sign=1.0):
    """x [B, N, H, D] and positions [B or 1, N, A] -> (turned x in 64 bits, |lo| + |hi| of every value)"""
    x, pos = x.double().cpu(), pos.double().cpu()
    y, size, P, j = x.clone(), torch.zeros_like(x), sum(sections), 0
    for a, n in enumerate(sections):
        for i in range(n):
            ang = sign * pos[..., a] * base ** (-(j / P) if shared else -(i / n))
            c, s = ang.cos()[..., None], ang.sin()[..., None]
            lo, hi = (2 * j, 2 * j + 1) if interleaved else (j, j + P)
            y[..., lo] = x[..., lo] * c - x[..., hi] * s
            y[..., hi] = x[..., hi] * c + x[..., lo] * s
            size[..., lo] = size[..., hi] = x[..., lo].abs() + x[..., hi].abs()
            j += 1
    return y, size


def close(got, want, size):
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double().cpu() - want).abs()
    tol = half * want.abs() + 6e-7 * (1 + half) * size + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert (off <= tol).all(), (float((off - tol).max()), got.dtype)


SHAPES = [  # (B, N, H, D, sections)
    (1, 1, 1, 2, (1,)), (8, 1, 8, 64, (8, 12, 12)), (2, 713, 5, 80, (16, 18)), (1, 9, 3, 40, (6, 7, 7)), (2, 33, 1, 256, (40, 44, 44)),
    (3, 5, 2, 6, (1, 0, 1)), (1, 3000, 2, 32, (4, 6, 6)), (1, 2, 700, 128, (10, 20, 30)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,N,H,D,sections", SHAPES)
def test_forward_and_gradient_match_the_definition(B, N, H, D, sections, dtype):
    from combo_avs_amd.ops.rotary import rotary_axes
    gen = torch.Generator().manual_seed(B * 7 + N + D)
    x = torch.randn(B, N, H, D, generator=gen).to(dtype).cuda().requires_grad_(True)
    dy = torch.randn(B, N, H, D, generator=gen).to(dtype).cuda()
    for interleaved, shared, per_batch, kind in ((False, False, False, torch.float32), (True, True, True, torch.int32),
                                                 (False, True, True, torch.int64), (True, False, False, torch.float64)):
        pos = torch.randint(-1_000_000, 1_000_000, (B if per_batch else 1, N, len(sections)), generator=gen).to(kind)
        if kind == torch.float64:
            pos = pos / 7
        p = (pos if per_batch else pos[0]).cuda()
        y = rotary_axes(x, p, sections, 10000.0, interleaved, shared)
        (dx,) = torch.autograd.grad(y, x, dy)
        assert y.is_contiguous() and y.dtype == dtype and dx.shape == x.shape
        close(y.detach(), *defined(x.detach(), pos, sections, 10000.0, interleaved, shared))
        close(dx, *defined(dy, pos, sections, 10000.0, interleaved, shared, -1.0))


def test_gradient_agrees_with_differences():
    from combo_avs_amd.ops.rotary import rotary_axes
    gen = torch.Generator().manual_seed(3)
    x, w, d = (torch.randn(1, 5, 2, 12, generator=gen).cuda() for _ in range(3))
    pos = torch.rand(5, 2, generator=gen).cuda() * 40
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad((rotary_axes(xg, pos, (2, 3)) * w).sum(), xg)
    # the op is linear: a difference over a step of 1 has no truncation error, only ~120 fp32 roundings of values of order 1
    diff = ((rotary_axes(x + d, pos, (2, 3)) - rotary_axes(x - d, pos, (2, 3))) * w).double().sum() / 2
    assert abs(float((g * d).double().sum() - diff)) < 120 * 4 * 2.0 ** -24 * 4


def test_strided_and_misaligned_inputs():
    from combo_avs_amd.ops.rotary import rotary_axes
    gen = torch.Generator().manual_seed(5)
    B, N, H, D = 2, 37, 3, 16
    pos = torch.randint(0, 50, (N, 2), generator=gen).cuda()
    fused = torch.randn(B, N, 3, H, D, generator=gen).cuda().bfloat16()
    flat = torch.randn(B * N * H * D + 1, generator=gen).cuda().bfloat16()
    views = [fused[:, :, 1], torch.randn(B, H, N, D, generator=gen).cuda().transpose(1, 2), torch.randn(B, N, H, D + 3, generator=gen).cuda()[..., 1:D + 1],
             torch.randn(B, N, D, H, generator=gen).cuda().transpose(2, 3), flat[1:].view(B, N, H, D), torch.randn(1, N, 1, D, generator=gen).cuda().expand(B, N, H, D)]
    for x in views:
        for interleaved in (False, True):
            y = rotary_axes(x, pos, (3, 4), 100.0, interleaved)
            assert torch.equal(y, rotary_axes(x.clone(memory_format=torch.contiguous_format), pos, (3, 4), 100.0, interleaved))
    wide = torch.randint(0, 50, (2, N, B), generator=gen).cuda()  # positions in another order of dimensions
    assert torch.equal(rotary_axes(views[0], wide.permute(2, 1, 0), (3, 4)), rotary_axes(views[0], wide.permute(2, 1, 0).contiguous(), (3, 4)))


def test_empty_no_pairs_and_zero_positions():
    from combo_avs_amd.ops.rotary import grid_positions, rotary_axes
    x = torch.randn(2, 6, 2, 8, device="cuda")
    assert torch.equal(rotary_axes(x, torch.zeros(6, 3, device="cuda"), (1, 1, 2)), x)
    assert torch.equal(rotary_axes(x, torch.ones(6, 1, device="cuda"), (0,)), x)
    e = torch.empty(0, 6, 2, 8, device="cuda", requires_grad=True)
    y = rotary_axes(e, torch.zeros(6, 1, device="cuda"), (2,))
    assert y.shape == e.shape and torch.autograd.grad(y.sum(), e)[0].shape == e.shape
    g = grid_positions(2, 3, 4, device="cuda")
    assert g.shape == (24, 3) and g[-1].tolist() == [1, 2, 3] and g[4].tolist() == [0, 1, 0]


def test_side_stream_and_graph_replays():
    from combo_avs_amd.ops.rotary import rotary_axes
    x = torch.randn(2, 100, 4, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    pos, dy = torch.rand(100, 2, device="cuda") * 50, torch.randn(2, 100, 4, 32, device="cuda").bfloat16()

    def step():
        y = rotary_axes(x, pos, (8, 8))
        return y.detach(), torch.autograd.grad(y, x, dy)[0]
    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(2, 100, 4, 32, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), held))
