"""Cases for timing the decoder-memory operators: group norm with an activation on channels-last maps, rotary positions
over several axes, and cross attention to encoder states of another length.

`run` computes an operator from elementary torch operations in 32 bits (`own` False) or calls the package's own entry
point (`own` True) on the same inputs; `exact` gives the same outputs from the definition in 64 bits."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WIDTH = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one frame's coarsest decoder level (224 / 32 = 7) while serving: the launch is what counts
        dict(name="norm_frame", op="norm", train=False, type="bf16", batch=1, channels=256, groups=32, height=7, width=7, act="silu"),
        # an image of no round size, a width that no power of two divides, exact GELU
        dict(name="norm_odd", op="norm", train=True, type="fp16", batch=3, channels=60, groups=6, height=117, width=93, act="gelu"),
        # the stride-4 maps of 8 clips x 5 frames at 224 x 224, in training
        dict(name="norm_clips", op="norm", train=True, type="bf16", batch=40, channels=256, groups=32, height=56, width=56, act="silu"),
        # one new token per sequence: the smallest call
        dict(name="rotary_token", op="rotary", train=False, type="bf16", batch=8, tokens=1, heads=8, dim=64, axes="8,12,12",
             interleaved=False, shared=False, far=True),
        # a cropped image's tokens with an unrotated rest of each head, pairs next to each other, one ladder over both axes
        dict(name="rotary_crop", op="rotary", train=False, type="fp16", batch=2, tokens=713, heads=5, dim=80, axes="16,18",
             interleaved=True, shared=True, far=False),
        # 8 clips x 5 frames of the stride-4 map as tokens of 8 heads x 32, in training
        dict(name="rotary_clips", op="rotary", train=True, type="bf16", batch=8, tokens=15680, heads=8, dim=32, axes="4,6,6",
             interleaved=False, shared=False, far=False),
        # one query token over a frame's stride-8 states, 8 heads x 32: the smallest call
        dict(name="cross_token", op="cross", train=False, type="bf16", batch=4, heads=8, groups=1, dim=32, queries=1, keys=784,
             ragged=False, blocked="none"),
        # single tokens of 16 sequences over long states of ragged length, four query heads to a key head
        dict(name="cross_token_long", op="cross", train=False, type="bf16", batch=16, heads=8, groups=4, dim=128, queries=1, keys=16384,
             ragged=True, blocked="none"),
        # the decoder's 100 queries over 40 frames' stride-8 maps under the masks predicted per query, in training
        dict(name="cross_queries", op="cross", train=True, type="bf16", batch=40, heads=8, groups=1, dim=32, queries=100, keys=784,
             ragged=False, blocked="query"),
        # image tokens that look at a short padded sequence (an utterance, a caption), in training
        dict(name="cross_short", op="cross", train=True, type="fp16", batch=4, heads=10, groups=1, dim=64, queries=4096, keys=77,
             ragged=True, blocked="none"),
        # image tokens over the memory of several frames, odd lengths, serving
        dict(name="cross_frames", op="cross", train=False, type="bf16", batch=2, heads=16, groups=1, dim=64, queries=4099, keys=15680,
             ragged=False, blocked="none"),
        # the largest: long queries and long states, wide heads, in training
        dict(name="cross_long", op="cross", train=True, type="bf16", batch=4, heads=16, groups=1, dim=128, queries=4096, keys=4096,
             ragged=False, blocked="none"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "cross", "cross"])
    train = rng.random() < 0.5
    if op == "norm":
        groups = rng.choice([1, 4, 6, 8, 16, 32])
        per = rng.choice([1, 2, 3, 4, 8, 10, 16])
        channels = groups * per
        height, width = _log(rng, 2, 160), _log(rng, 2, 160)  # (one or two values in a group have a gradient of rounding only)
        batch = _log(rng, 1, 64)
        while batch > 1 and batch * channels * height * width > 32_000_000:
            batch //= 2
        return dict(op=op, train=train, type=rng.choice(["bf16", "fp16", "fp32"]), batch=batch, channels=channels, groups=groups,
                    height=height, width=width, act=rng.choice(["none", "relu", "silu", "gelu"]))
    if op == "rotary":
        dim, axes = rng.choice([(32, "4,6,6"), (32, "8,8"), (64, "8,12,12"), (64, "32"), (80, "16,18"), (40, "6,7,7"), (128, "16,24,24"),
                                (96, "16,16,16"), (128, "10,20,30")])
        tokens, heads, batch = _log(rng, 1, 20000), _log(rng, 1, 32), _log(rng, 1, 32)
        while batch > 1 and batch * tokens * heads * dim > 32_000_000:
            batch //= 2
        tokens = max(1, min(tokens, 32_000_000 // (batch * heads * dim)))
        return dict(op=op, train=train, type=rng.choice(["bf16", "fp16", "fp32"]), batch=batch, tokens=tokens, heads=heads, dim=dim,
                    axes=axes, interleaved=rng.random() < 0.5, shared=rng.random() < 0.5, far=rng.random() < 0.3)
    kind = rng.choice(["token", "queries", "image", "long"])
    queries, keys = {"token": lambda: (_log(rng, 1, 8), _log(rng, 1, 32768)), "queries": lambda: (_log(rng, 16, 300), _log(rng, 49, 16384)),
                     "image": lambda: (_log(rng, 256, 8192), _log(rng, 16, 512)),
                     "long": lambda: (_log(rng, 512, 4096), _log(rng, 512, 4096))}[kind]()
    dim, heads, groups = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128]), _log(rng, 1, 16), rng.choice([1, 1, 1, 2, 4, 8])
    batch = _log(rng, 1, 64)

    def much(b):
        return (b * heads * groups * queries * keys > 1_000_000_000 or b * heads * dim * (groups * queries + 2 * keys) > 400_000_000)
    while much(batch) and batch > 1:
        batch //= 2
    while much(batch) and groups > 1:
        groups //= 2
    while much(batch) and heads > 1:
        heads //= 2
    return dict(op=op, train=train, type=rng.choice(["bf16", "fp16"]), batch=batch, heads=heads, groups=groups, dim=dim, queries=queries,
                keys=keys, ragged=rng.random() < 0.5, blocked=rng.choice(["none", "none", "query", "key"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, dev = TYPES[case["type"]], "cuda"

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, device=dev, generator=gen).to(dtype)
    s = {"case": case}
    if case["op"] == "norm":
        B, C, H, W = case["batch"], case["channels"], case["height"], case["width"]
        # a convolution's output: channels of different scale and offset
        offset, size = torch.randn(C, device=dev, generator=gen), torch.rand(C, device=dev, generator=gen) + 0.5
        x = (torch.randn(B, H, W, C, device=dev, generator=gen) * size + offset).to(dt)
        s["x"] = x.permute(0, 3, 1, 2)
        s["weight"] = torch.rand(C, device=dev, generator=gen) + 0.5
        s["bias"] = torch.randn(C, device=dev, generator=gen) * 0.5
        if case["train"]:
            s["dy"] = normal(B, H, W, C).permute(0, 3, 1, 2)
            leaves = [s["x"], s["weight"], s["bias"]]
    elif case["op"] == "rotary":
        B, N, A = case["batch"], case["tokens"], len(case["axes"].split(","))
        s["x"] = normal(B, N, case["heads"], case["dim"])
        if case["far"]:  # tokens far into a long stream, each sequence at its own place
            s["pos"] = torch.randint(0, 1_000_000, (B, N, A), device=dev, generator=gen, dtype=torch.int32)
        else:  # the places of a grid, the last axis running fastest
            side = max(1, int(round(N ** (1.0 / A))))
            n = torch.arange(N, device=dev)
            s["pos"] = torch.stack([(n // side ** (A - 1 - a)) % (side if a else N) for a in range(A)], -1).float()
        if case["train"]:
            s["dy"] = normal(*s["x"].shape)
            leaves = [s["x"]]
    else:
        B, H, G, D, Lq, Lk = (case[k] for k in ("batch", "heads", "groups", "dim", "queries", "keys"))
        s["q"], s["k"], s["v"] = normal(B, Lq, H * G, D), normal(B, Lk, H, D), normal(B, Lk, H, D)
        s["lengths"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint((Lk + 3) // 4, Lk + 1, (B,), device=dev, generator=gen, dtype=torch.int32)
        s["blocked"] = None
        if case["blocked"] == "query":  # the masks of a segmentation head: a query sees its region, a few see nothing
            s["blocked"] = torch.rand(B, 1, Lq, Lk, device=dev, generator=gen) < 0.6
            s["blocked"] |= torch.rand(B, 1, Lq, 1, device=dev, generator=gen) < 0.02
        elif case["blocked"] == "key":
            s["blocked"] = torch.rand(B, 1, 1, Lk, device=dev, generator=gen) < 0.3
        if case["train"]:
            s["dy"] = normal(B, Lq, H * G, D)
            leaves = [s["q"], s["k"], s["v"]]
    if case["train"]:
        s["leaves"] = [t.requires_grad_(True) for t in leaves]
    return s


def run(state):
    case = state["case"]
    if own:
        y = _call(case, state)
        if not case["train"]:
            return y
        return [y.detach()] + list(torch.autograd.grad(y, state["leaves"], state["dy"]))
    with torch.no_grad():
        return {"norm": _norm, "rotary": _rotary, "cross": _cross}[case["op"]](case, state)


def _call(case, s):
    if case["op"] == "norm":
        from combo_avs_amd.ops.groupnorm import group_norm_act
        return group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], eps=1e-5, activation=case["act"])
    if case["op"] == "rotary":
        from combo_avs_amd.ops.rotary import rotary_axes
        return rotary_axes(s["x"], s["pos"], _axes(case), base=10000.0, interleaved=case["interleaved"], shared_ladder=case["shared"])
    from combo_avs_amd.ops.cross_attention import cross_attention
    return cross_attention(s["q"], s["k"], s["v"], kv_lengths=s["lengths"], blocked=s["blocked"])


def _axes(case):
    return tuple(int(n) for n in case["axes"].split(","))


# ---- plain forms ----------------------------------------------------------------------------------------------------------

def _phi(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z * _phi(z) if act == "gelu" else z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return _phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _norm(case, s):
    B, C, H, W = s["x"].shape
    G, dt = case["groups"], s["x"].dtype
    x = s["x"].permute(0, 2, 3, 1).float().reshape(B, H * W, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean((1, 3), keepdim=True) + 1e-5)
    xh = (x - mean) * rstd
    w, b = s["weight"].view(G, C // G), s["bias"].view(G, C // G)
    z = xh * w + b

    def out(t):
        return t.reshape(B, H, W, C).to(dt).permute(0, 3, 1, 2)
    y = out(_act(z, case["act"]))
    if not case["train"]:
        return y
    dz = s["dy"].permute(0, 2, 3, 1).float().reshape(B, H * W, G, C // G) * _act_slope(z, case["act"])
    dw, db = (dz * xh).sum((0, 1)).reshape(C), dz.sum((0, 1)).reshape(C)
    dxh = dz * w
    dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
    return [y, out(dx), dw, db]


def _turns(case, pos):
    """angles [..., pairs] in 64 bits: axis a turns its own pairs"""
    sections, out, done = _axes(case), [], 0
    for a, n in enumerate(sections):
        i = torch.arange(n, device=pos.device, dtype=torch.float64)
        i = (i + done) / sum(sections) if case["shared"] else i / n
        out.append(pos[..., a:a + 1].double() * 10000.0 ** -i)
        done += n
    return torch.cat(out, -1)


def _rotary(case, s):
    a = _turns(case, s["pos"])
    cos, sin = a.cos().float().unsqueeze(-2), a.sin().float().unsqueeze(-2)
    P, dt = a.shape[-1], s["x"].dtype

    def turn(x, sin):
        x = x.float()
        if case["interleaved"]:
            lo, hi = x[..., 0:2 * P:2], x[..., 1:2 * P:2]
            pairs = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], -1).flatten(-2)
        else:
            lo, hi = x[..., :P], x[..., P:2 * P]
            pairs = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
        return torch.cat([pairs, x[..., 2 * P:]], -1).to(dt)
    y = turn(s["x"], sin)
    return [y, turn(s["dy"], -sin)] if case["train"] else y


def _cross(case, s):
    B, H, G, D, Lq, Lk = (case[k] for k in ("batch", "heads", "groups", "dim", "queries", "keys"))
    dt, scale = s["q"].dtype, D ** -0.5

    def rows(t):  # [B, Lq, H G, D] -> [B, H, G Lq, D]
        return t.float().view(B, Lq, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Lq, D)

    def back(t):
        return t.view(B, H, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, H * G, D).to(dt)
    q, k, v = rows(s["q"]), s["k"].float().transpose(1, 2).contiguous(), s["v"].float().transpose(1, 2).contiguous()
    p = (q @ k.transpose(2, 3).contiguous()).mul_(scale).view(B, H, G, Lq, Lk)
    if s["lengths"] is not None:
        p.masked_fill_((torch.arange(Lk, device=p.device) >= s["lengths"][:, None])[:, None, None, None], float("-inf"))
    if s["blocked"] is not None:
        p.masked_fill_(s["blocked"].unsqueeze(2), float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill_(top == float("-inf"), 0)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total.masked_fill_(total == 0, 1))  # a query that sees nothing: zeros
    p = p.view(B, H, G * Lq, Lk)
    y = back(p @ v)
    if not case["train"]:
        return y
    dy = rows(s["dy"])
    dv = p.transpose(2, 3).contiguous() @ dy
    ds = dy @ v.transpose(2, 3).contiguous()
    ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p)
    dq, dk = (ds @ k).mul_(scale), (ds.transpose(2, 3).contiguous() @ q).mul_(scale)
    return [y, back(dq), dk.transpose(1, 2).to(dt).contiguous(), dv.transpose(1, 2).to(dt).contiguous()]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    e, train = WIDTH[case["type"]], case["train"]
    if case["op"] == "norm":
        n = case["batch"] * case["channels"] * case["height"] * case["width"]
        return {"bytes": n * e * (4 if train else 2) + 4 * case["channels"] * (4 if train else 2), "flops": n * (40 if train else 12)}
    if case["op"] == "rotary":
        places = case["batch"] * case["tokens"]
        n = places * case["heads"] * case["dim"]
        axes = len(_axes(case))
        return {"bytes": n * e * (4 if train else 2) + 4 * axes * (places if case["far"] else case["tokens"]), "flops": n * (6 if train else 3)}
    B, H, G, D, Lq, Lk = (case[k] for k in ("batch", "heads", "groups", "dim", "queries", "keys"))
    seen = 0.625 * Lk if case["ragged"] else Lk  # the mean of the lengths drawn
    q, kv = B * Lq * H * G * D, int(2 * B * seen * H * D)
    masks = {"none": 0, "key": B * Lk, "query": B * Lq * Lk}[case["blocked"]]
    scores = B * H * G * Lq * seen
    if not train:
        return {"bytes": (2 * q + kv) * e + masks, "flops": int(4 * scores * D)}
    return {"bytes": (4 * q + kv) * e + 2 * B * Lk * H * D * e + masks, "flops": int(14 * scores * D)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items() if k != "leaves"}
    return {"norm": _exact_norm, "rotary": _exact_rotary, "cross": _exact_cross}[case["op"]](case, s)


def _exact_norm(case, s):
    f = torch.nn.functional
    x, w, b = (s[k].requires_grad_(case["train"]) for k in ("x", "weight", "bias"))
    z = f.group_norm(x.contiguous(), case["groups"], w, b, 1e-5)
    y = {"none": lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu}[case["act"]](z)
    if not case["train"]:
        return y
    return [y.detach()] + list(torch.autograd.grad(y, (x, w, b), s["dy"]))


def _exact_rotary(case, s):
    sections = _axes(case)
    pairs = sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    rate = [10000.0 ** (-j / pairs) if case["shared"] else 10000.0 ** (-(j - sum(sections[:a])) / sections[a]) for j, a in enumerate(axis)]

    def turned(x, sign):
        y = x.clone()
        for j in range(pairs):
            lo, hi = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + pairs)
            z = torch.polar(torch.ones_like(s["pos"][..., 0].double()), sign * rate[j] * s["pos"][..., axis[j]].double()).unsqueeze(-1)
            w = torch.complex(x[..., lo], x[..., hi]) * z
            y[..., lo], y[..., hi] = w.real, w.imag
        return y
    y = turned(s["x"], 1.0)
    return [y, turned(s["dy"], -1.0)] if case["train"] else y


def _exact_cross(case, s):
    G, D = case["groups"], case["dim"]
    y = torch.zeros_like(s["q"])
    grads = [torch.zeros_like(s[k]) for k in ("q", "k", "v")] if case["train"] else None
    for b in range(case["batch"]):
        n = int(s["lengths"][b]) if s["lengths"] is not None else case["keys"]
        for h in range(case["heads"]):
            hs = slice(h * G, (h + 1) * G)
            q, k, v = (t.detach().requires_grad_(case["train"]) for t in (s["q"][b, :, hs], s["k"][b, :n, h], s["v"][b, :n, h]))
            scores = torch.matmul(q, k.t()) / math.sqrt(D)  # [Lq, G, n]
            open_ = torch.ones_like(scores, dtype=torch.bool)
            if s["blocked"] is not None:
                open_ = open_ & ~s["blocked"][b, 0, :, None, :n]
            some = open_.any(-1, keepdim=True)
            weights = torch.softmax(scores.masked_fill(~open_ & some, float("-inf")), -1) * some
            o = torch.matmul(weights, v)
            y[b, :, hs] = o.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["dy"][b, :, hs])
                grads[0][b, :, hs], grads[1][b, :n, h], grads[2][b, :n, h] = dq, dk, dv
    return [y] + grads if case["train"] else y
