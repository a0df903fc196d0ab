"""Cross attention (csrc/cross_attention.hip, ops/cross_attention.py) against the formulas in 64 bits on the same operands.

Tolerances, derived (h: half a step of the type, u = 2^-24).  A score is a sum of D products, off by at most E = (D + 4) u scale sum |q k|
(order of summation free, exp2's argument included), so a probability is off by 2 E + 8 u relative, and by h where it is rounded for the
second product.  With N = sum_j p_j |v_j|:
    out:   h |o| + (h + 2 E + 16 u) N
    delta: sum_d |do_d| tol(o_d);   dp: (D + 4) u sum |do v|
    ds:    h |ds| + (2 E + 16 u) |ds| + p (tol(delta) + tol(dp))
    dq:    h |dq| + scale sum_j (tol(ds_j) + n u |ds_j|) |k_j|, dk likewise over the rows;  dv: h |dv| + sum_r (h + 2 E + 16 u + n u) p |do|
n: the length of the last sums.  fp16 keeps nothing under 2^-25, which every rounded p, ds and result adds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def defined(q, k, v, lengths, blocked, scale, dout):
    """-> results and tolerances [out, dq, dk, dv] in 64 bits on the CPU"""
    dt = q.dtype
    h, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == torch.float16 else 0.0
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1:3]
    G = Hq // Hk
    Q, K, V, DO = (t.detach().double().cpu().transpose(1, 2) for t in (q, k, v, dout))  # [B, H, L, D]
    shut = torch.zeros(B, Hq, Lq, Lk, dtype=torch.bool)
    if lengths is not None:
        shut |= (torch.arange(Lk) >= lengths.cpu().clamp(0, Lk)[:, None])[:, None, None]
    if blocked is not None:
        shut |= blocked.cpu()
    gone = shut.all(2).all(1)  # states that nobody sees may hold anything
    K, V = (torch.where(gone[:, None, :, None], torch.zeros_like(t), t) for t in (K, V))
    Kg, Vg = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    s = scale * Q @ Kg.transpose(2, 3)
    E = (D + 4) * U * scale * (Q.abs() @ Kg.abs().transpose(2, 3)) + 4 * U * s.abs()
    E = E.masked_fill(shut, 0).amax(-1, keepdim=True)
    s = s.masked_fill(shut, float("-inf"))
    none = shut.all(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
    o = p @ Vg
    r = 2 * E + 16 * U
    t_o = h * o.abs() + (h + r) * (p @ Vg.abs()) + tiny * (1 + (~shut).double() @ Vg.abs())
    dp = DO @ Vg.transpose(2, 3)
    delta = (DO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    t_ds = (h + r) * ds.abs() + p * ((DO.abs() * t_o).sum(-1, keepdim=True) + (D + 4) * U * (DO.abs() @ Vg.abs().transpose(2, 3))) + tiny
    t_ds = t_ds.masked_fill(shut, 0)
    dq = scale * ds @ Kg
    t_dq = h * dq.abs() + scale * (t_ds + Lk * U * ds.abs()) @ Kg.abs() + tiny

    def group(t):
        return t.view(B, Hk, G, Lk, D).sum(2)
    dk, dv = group(scale * ds.transpose(2, 3) @ Q), group(p.transpose(2, 3) @ DO)
    n = Lq * G
    t_dk = h * dk.abs() + group(scale * (t_ds + n * U * ds.abs()).transpose(2, 3) @ Q.abs()) + tiny
    t_dv = h * dv.abs() + group((p * (h + r + n * U) + tiny * (p > 0)).transpose(2, 3) @ DO.abs()) + tiny
    return [t.transpose(1, 2) for t in (o, dq, dk, dv)], [t.transpose(1, 2) for t in (t_o, t_dq, t_dk, t_dv)]


def check(q, k, v, lengths=None, blocked=None, scale=None, dout=None):
    from combo_avs_amd.ops.cross_attention import cross_attention
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(9)).to(q.dtype).cuda() if dout is None else dout
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, lengths, blocked, scale)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, dout))
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v, lengths, blocked, scale), got[0])
    want, tol = defined(q, k, v, lengths, blocked, scale or q.shape[3] ** -0.5, dout)
    for name, a, b, t in zip(("out", "dq", "dk", "dv"), got, want, tol):
        off = (a.double().cpu() - b).abs()
        assert (off <= t + 1e-30).all(), (name, float((off / (t + 1e-30)).max()), float(off.max()))
    return got


def made(B, Lq, Lk, Hq, Hk, D, dtype, seed=0, size=1.0):
    gen = torch.Generator().manual_seed(seed + B * 31 + Lq + Lk * 7 + D)
    return [(size * torch.randn(B, L, H, D, generator=gen)).to(dtype).cuda() for L, H in ((Lq, Hq), (Lk, Hk), (Lk, Hk))]


SHAPES = [  # (B, Lq, Lk, Hq, Hk, D): one token, short and long states, grouped heads, head dimensions inside a tile, split keys, split rows
    (1, 1, 1, 1, 1, 8), (2, 1, 784, 8, 8, 32), (2, 1, 1500, 8, 2, 128), (3, 5, 77, 4, 2, 40), (2, 33, 129, 2, 1, 64), (1, 300, 65, 3, 3, 128),
    (2, 100, 784, 2, 2, 32), (1, 257, 1025, 2, 2, 80), (1, 4097, 33, 1, 1, 16), (1, 40, 5000, 1, 1, 64), (1, 2, 4100, 16, 1, 96), (2, 700, 300, 8, 1, 56),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hk,D", SHAPES)
def test_matches_the_formulas(B, Lq, Lk, Hq, Hk, D, dtype):
    q, k, v = made(B, Lq, Lk, Hq, Hk, D, dtype)
    check(q, k, v)
    gen = torch.Generator().manual_seed(Lk)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen, dtype=torch.int32)
    lengths[0] = min(Lk, 1)
    check(q, k, v, lengths=lengths.cuda())
    per_query = torch.rand(B, 1, Lq, Lk, generator=gen) < 0.7
    per_query |= torch.rand(B, 1, Lq, 1, generator=gen) < 0.2  # rows that see nothing
    check(q, k, v, blocked=per_query.cuda(), lengths=lengths.cuda().long())
    per_head = torch.rand(1, Hq, Lq, Lk, generator=gen) < 0.5
    check(q, k, v, blocked=per_head.cuda(), scale=0.3)
    check(q, k, v, blocked=(torch.rand(B, 1, 1, Lk, generator=gen) < 0.5).cuda())


@pytest.mark.parametrize("Lq,Hq,Hk", [(1, 4, 4), (5, 4, 2), (150, 2, 2)])
def test_lengths_at_every_border(Lq, Hq, Hk):
    q, k, v = made(8, Lq, 140, Hq, Hk, 64, torch.bfloat16)
    for group in ([0, 1, 2, 31, 32, 33, 63, 64], [65, 95, 96, 97, 127, 128, 129, 140], [-3, 1000, 139, 0, 0, 0, 0, 0]):
        check(q, k, v, lengths=torch.tensor(group, dtype=torch.int32).cuda())


def test_states_nobody_sees_may_hold_anything():
    from combo_avs_amd.ops.cross_attention import cross_attention
    for Lq in (1, 70):
        q, k, v = made(2, Lq, 200, 4, 2, 64, torch.bfloat16)
        lengths = torch.tensor([150, 37], dtype=torch.int32).cuda()
        blocked = (torch.arange(200) % 5 == 0).view(1, 1, 1, 200).cuda()
        dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
        res = []
        for filler in (0.0, float("nan"), float("inf"), 3e38):
            kk, vv = k.clone(), v.clone()
            for t in (kk, vv):
                t[:, ::5] = filler
                for b in range(2):
                    t[b, int(lengths[b]):] = filler
            leaves = [t.requires_grad_(True) for t in (q.clone(), kk, vv)]
            out = cross_attention(*leaves, lengths, blocked)
            res.append([out.detach()] + list(torch.autograd.grad(out, leaves, dout)))
        for other in res[1:]:
            assert all(torch.equal(a, b) for a, b in zip(res[0], other))


def test_rows_that_see_nothing_and_rows_that_see_one_key():
    q, k, v = made(1, 64, 100, 2, 2, 32, torch.bfloat16)
    blocked = torch.ones(1, 1, 64, 100, dtype=torch.bool)
    out, dq, dk, dv = check(q, k, v, blocked=blocked.cuda())
    assert not out.any() and not dq.any() and not dk.any() and not dv.any()
    blocked[0, 0, torch.arange(64), torch.arange(64)] = False
    out, dq, dk, dv = check(q, k, v, blocked=blocked.cuda())
    assert torch.equal(out, v[:, :64]) and not dq.any() and not dk.any()  # one key: p = 1, nothing to learn from its score


def test_large_scores():
    """scores of +-100: one-hot rows, underflow on the other side"""
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = made(2, 40, 300, 2, 2, 64, dtype, size=3.5)
        got = check(q, k, v)
        assert all(torch.isfinite(t.float()).all() for t in got)
    q, k, v = made(1, 3, 260, 4, 2, 128, torch.bfloat16, size=3.0)
    check(q, k, v + 20)  # values with an offset: delta = do . o cancels against do . v


def test_strides_orders_and_alignment():
    from combo_avs_amd.ops.cross_attention import cross_attention
    gen = torch.Generator().manual_seed(2)
    B, Lq, Lk, H, D = 2, 50, 90, 4, 32
    kv = torch.randn(B, Lk, 2, H, D, generator=gen).bfloat16().cuda()
    q = torch.randn(B, H, Lq, D, generator=gen).bfloat16().cuda().transpose(1, 2)
    k, v = kv.unbind(2)
    check(q, k, v)
    check(q[:, ::2], k[:, 1::3], v[:, 1::3])
    flat = torch.randn(B * Lk * H * D + 3, generator=gen).bfloat16().cuda()[3:].view(B, Lk, H, D)
    check(q, flat, v)
    wide = torch.randn(B, Lk, H, D + 1, generator=gen).bfloat16().cuda()[..., 1:]
    check(q, wide, torch.randn(B, Lk, D, H, generator=gen).bfloat16().cuda().transpose(2, 3))
    check(q, k[:1].expand(B, Lk, H, D), v[:, :, :1].expand(B, Lk, H, D))
    mask = torch.rand(Lk, Lq, generator=gen) < 0.4
    check(q, k, v, blocked=mask.cuda().t()[None, None])
    check(q, k, v, blocked=(torch.rand(B, H, Lq, Lk + 5, generator=gen) < 0.4).cuda()[..., 3:Lk + 3])
    check(q, k, v, blocked=(torch.rand(B, H, 1, Lk, generator=gen) < 0.4).cuda().expand(B, H, Lq, Lk))
    o = cross_attention(q.detach().requires_grad_(True), k, v)
    o.sum().backward()  # an expanded gradient; only q asks


def test_frozen_states_and_partial_gradients():
    from combo_avs_amd.ops.cross_attention import cross_attention
    q, k, v = made(2, 30, 100, 2, 2, 64, torch.float16)
    dout = torch.randn_like(q)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(cross_attention(*full), full, dout)
    for mask in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((q, k, v))]
        ask = [t for t in leaves if t.requires_grad]
        got = torch.autograd.grad(cross_attention(*leaves), ask, dout)
        assert all(torch.equal(a, b) for a, b in zip(got, [w for i, w in enumerate(want) if mask >> i & 1]))


def test_empty_sizes():
    from combo_avs_amd.ops.cross_attention import cross_attention
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = (torch.randn(B, L, 2, 16, device="cuda").bfloat16().requires_grad_(True) for L in (Lq, Lk, Lk))
        out = cross_attention(q, k, v)
        grads = torch.autograd.grad(out.sum(), (q, k, v))
        assert out.shape == q.shape and not out.any() and all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))
        with torch.no_grad():
            assert not cross_attention(q, k, v).any()


def test_gradient_agrees_with_differences():
    from combo_avs_amd.ops.cross_attention import cross_attention
    q, k, v = made(1, 6, 20, 2, 1, 16, torch.float16)
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).half().cuda()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*leaves), leaves, w)
    h = 2.0 ** -4
    for i in range(3):
        step = torch.randint(0, 2, leaves[i].shape, generator=torch.Generator().manual_seed(i)).half().cuda() * 2 - 1  # exact in fp16 up to |x| = 64
        at = [[t.detach() + (s * h * step if j == i else 0) for j, t in enumerate((q, k, v))] for s in (1, -1)]
        moved = (at[0][i].double() - at[1][i].double()) / 2  # what the rounded inputs really moved by
        diff = ((cross_attention(*at[0]).double() - cross_attention(*at[1]).double()) * w).sum() / 2
        got = (grads[i].double() * moved).sum()
        # 192 outputs of order 1, each off by at most 2 h = 2^-10 (two roundings), random signs: 14 * 2^-10 = 0.014, four times that;
        # truncation: a third derivative of order D^1.5 scale^3 = 1 per row along a step of +-1, h^3 / 6 * 192 = 0.008
        assert abs(float(got - diff)) < 0.064, (i, float(got), float(diff))


def test_runs_repeat_bit_for_bit_on_streams_and_in_graphs():
    from combo_avs_amd.ops.cross_attention import cross_attention
    for B, Lq, Lk in ((2, 1, 900), (2, 200, 333)):
        q, k, v = made(B, Lq, Lk, 4, 2, 64, torch.bfloat16)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
        lengths = torch.tensor([Lk, Lk // 2], dtype=torch.int32).cuda()
        blocked = (torch.rand(B, 1, Lq, Lk, generator=torch.Generator().manual_seed(5)) < 0.3).cuda()

        def step():
            out = cross_attention(*leaves, lengths, blocked)
            return [out.detach()] + list(torch.autograd.grad(out, leaves, dout))
        eager = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(eager, other))
        graph, twin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        with torch.cuda.graph(twin, pool=graph.pool()):
            held2 = step()
        for seed in range(3):
            with torch.no_grad():
                q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
                lengths.copy_(torch.tensor([Lk // 3 + seed, Lk], dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(step(), held))
            twin.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(step(), held2))


@pytest.mark.parametrize("B,Lk,Hq,Hk,D", [(1, 9000, 2, 1, 128), (1, 17000, 3, 3, 64), (2, 1030, 4, 2, 16), (64, 4100, 8, 8, 8)])
def test_single_tokens_over_long_states(B, Lk, Hq, Hk, D):
    """shares of a row by the dozen, shares that a short sample leaves empty, and halved shares"""
    q, k, v = made(B, 1, Lk, Hq, Hk, D, torch.bfloat16)
    check(q, k, v)
    lengths = torch.randint(0, Lk + 1, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32)
    check(q, k, v, lengths=lengths.cuda(), blocked=(torch.rand(B, 1, 1, Lk, generator=torch.Generator().manual_seed(Lk)) < 0.3).cuda())


@pytest.mark.parametrize("B,Lq,Lk,Hq,Hk,D,dtype", [(16, 129, 300, 8, 8, 32, torch.bfloat16), (16, 130, 161, 8, 8, 64, torch.float16), (16, 150, 100, 8, 8, 80, torch.bfloat16),
                                                   (32, 70, 77, 8, 4, 40, torch.float16), (16, 129, 130, 8, 8, 128, torch.bfloat16), (16, 129, 90, 8, 8, 128, torch.float16), (9, 1000, 31, 4, 4, 24, torch.bfloat16)])
def test_blocks_that_fill_the_chip(B, Lq, Lk, Hq, Hk, D, dtype):
    """at least 256 blocks of 128 rows, whose keys are not split"""
    q, k, v = made(B, Lq, Lk, Hq, Hk, D, dtype)
    gen = torch.Generator().manual_seed(D)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen, dtype=torch.int32)
    lengths[:3] = torch.tensor([Lk, 0, 1])
    check(q, k, v)
    check(q, k, v, lengths=lengths.cuda(), blocked=(torch.rand(B, 1, Lq, Lk, generator=gen) < 0.6).cuda())
    check(q, k, v, lengths=lengths.cuda(), blocked=(torch.rand(B, 1, 1, Lk, generator=gen) < 0.5).cuda())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Lq,Lk,D", [(8, 4, 512, 4, 64), (8, 4, 512, 16, 16), (2, 4, 512, 40, 128), (2, 4, 512, 300, 16), (8, 4, 8, 2000, 64), (1, 1, 300, 16384, 64),
                                            (16, 8, 512, 90, 128), (16, 8, 512, 40, 80), (16, 8, 512, 190, 64)])
def test_errors_are_those_of_two_roundings(B, H, Lq, Lk, D, dtype):
    """Root mean squares: a result carries its own rounding and that of one operand (p or ds), independent and as large where mantissas are spread
    alike: sqrt(2) times the error of rounding the exact result, and an eighth more for mantissas that are not."""
    from combo_avs_amd.ops.cross_attention import cross_attention
    gen = torch.Generator().manual_seed(Lk + D)
    q, k, v, dout = (torch.randn(B, L, H, D, generator=gen).to(dtype) for L in (Lq, Lk, Lk, Lq))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves)
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, dout.cuda()))
    want, _ = defined(q, k, v, None, None, D ** -0.5, dout)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        off, own = (a.double().cpu() - b).norm(), (b.to(dtype).double() - b).norm()
        assert off <= 1.125 * 2 ** 0.5 * own, (name, float(off / own))
