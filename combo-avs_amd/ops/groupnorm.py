"""GroupNorm (+ ReLU) on channels_last fp32 maps (csrc/groupnorm.hip): no NCHW round trip, channels_last in and out."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib


def usable(x, gn):
    return (x.is_cuda and x.dtype == torch.float32 and x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last)
            and x.shape[1] % 4 == 0 and x.shape[1] <= 1024 and gn.affine and not torch.is_autocast_enabled())


class _GroupNormNHWC(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, relu):
        B, C, H, W = x.shape
        lib = _lib.lib()
        slices = lib.combo_groupnorm_nhwc_slices(H * W)
        dev = x.device
        y = torch.empty_like(x)  # preserves channels_last
        mean = torch.empty(B, groups, device=dev, dtype=torch.float32)
        rstd = torch.empty(B, groups, device=dev, dtype=torch.float32)
        part = torch.empty(B * slices * C * 2, device=dev, dtype=torch.float32)
        _lib.check(lib.combo_groupnorm_nhwc_forward_f32(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), B, H * W, C, groups, eps,
                                                        1 if relu else 0, part.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                                        y.data_ptr(), _lib.current_stream()), "combo_groupnorm_nhwc_forward_f32")
        ctx.save_for_backward(x, y if relu else None, mean, rstd, weight)
        ctx.groups, ctx.relu = groups, relu
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, y, mean, rstd, weight = ctx.saved_tensors
        B, C, H, W = x.shape
        lib = _lib.lib()
        dev = x.device
        dy = dy.contiguous(memory_format=torch.channels_last)
        slices = lib.combo_groupnorm_nhwc_slices(H * W)
        part = torch.empty(B * slices * C * 2, device=dev, dtype=torch.float32)
        s12 = torch.empty(B * ctx.groups * 2 + B * C * 2, device=dev, dtype=torch.float32)
        dx = torch.empty_like(x)
        dgamma = torch.empty(C, device=dev, dtype=torch.float32)
        dbeta = torch.empty(C, device=dev, dtype=torch.float32)
        _lib.check(lib.combo_groupnorm_nhwc_backward_f32(dy.data_ptr(), x.data_ptr(), _lib.ptr(y), mean.data_ptr(), rstd.data_ptr(),
                                                         weight.data_ptr(), B, H * W, C, ctx.groups, 1 if ctx.relu else 0,
                                                         part.data_ptr(), s12.data_ptr(), dx.data_ptr(), dgamma.data_ptr(),
                                                         dbeta.data_ptr(), _lib.current_stream()), "combo_groupnorm_nhwc_backward_f32")
        return dx, dgamma, dbeta, None, None, None


def group_norm(x, gn, relu=False):
    """x: channels_last fp32 [B,C,H,W]; gn: nn.GroupNorm -> channels_last output (ReLU fused when asked)."""
    return _GroupNormNHWC.apply(x, gn.weight, gn.bias, gn.num_groups, gn.eps, relu)


# ---- group norm with an activation, any of the float types and any channel count (csrc/groupnorm_act.hip) ----

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
MAX_CHANNELS = 4096


def _channels_last(x):
    return torch.channels_last if x.dim() == 4 else torch.channels_last_3d


def _act_workspace(x, places, groups, code, backward):
    n = _lib.lib().combo_groupnorm_act_workspace(x.shape[0], places, x.shape[1], groups, code, backward)
    if n < 0:
        raise ValueError(f"group_norm_act: sizes the kernels do not take: {tuple(x.shape)}")
    return torch.empty(n, device=x.device, dtype=torch.float32) if n else None


def _act_forward(x, weight, bias, groups, eps, act, keep=False):
    """weight, bias: contiguous fp32 or None -> (y, mean and rstd [2, B, groups] for the backward pass or None)"""
    B, C, places = int(x.shape[0]), int(x.shape[1]), x.shape[2:].numel()
    y = torch.empty_like(x)  # (preserves channels_last)
    stats = torch.empty(2, B, groups, device=x.device, dtype=torch.float32) if keep else None
    if x.numel() == 0:
        return y, stats
    code, mean = _lib.FLOAT_TYPES[x.dtype], _lib.ptr(stats)
    with _lib.device_of(x) as stream:
        ws = _act_workspace(x, places, groups, code, 0)
        _lib.check(_lib.lib().combo_groupnorm_act_forward(x.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), B, places, C, groups, eps, act, code,
                                                          _lib.ptr(ws), mean, mean + 4 * B * groups if keep else 0, y.data_ptr(), stream),
                   "combo_groupnorm_act_forward")
    return y, stats


def _param(p):
    return None if p is None else p.float().contiguous()


def _as_given(dw, db, types):
    return [g if g is None or g.dtype == t else g.to(t) for g, t in zip((dw, db), types)]


class _GroupNormAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        ctx.groups, ctx.act, ctx.types = groups, act, [None if p is None else p.dtype for p in (weight, bias)]
        weight, bias = _param(weight), _param(bias)
        y, stats = _act_forward(x, weight, bias, groups, eps, act, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        B, C = x.shape[:2]
        dx = torch.empty_like(x)
        new = torch.zeros if x.numel() == 0 else torch.empty
        dw = new(C, device=x.device, dtype=torch.float32) if weight is not None and ctx.needs_input_grad[1] else None
        db = new(C, device=x.device, dtype=torch.float32) if bias is not None and ctx.needs_input_grad[2] else None
        if x.numel() == 0:
            return (dx, *_as_given(dw, db, ctx.types), None, None, None)
        dy = dy.contiguous(memory_format=_channels_last(x))
        code, base, places = _lib.FLOAT_TYPES[x.dtype], stats.data_ptr(), x.shape[2:].numel()
        with _lib.device_of(x) as stream:
            ws = _act_workspace(x, places, ctx.groups, code, 1)
            _lib.check(_lib.lib().combo_groupnorm_act_backward(dy.data_ptr(), x.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), base,
                                                               base + 4 * B * ctx.groups, B, places, C, ctx.groups, ctx.act, code,
                                                               ws.data_ptr(), dx.data_ptr(), _lib.ptr(dw), _lib.ptr(db), stream),
                       "combo_groupnorm_act_backward")
        return (dx, *_as_given(dw, db, ctx.types), None, None, None)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, activation="none"):
    """act(GroupNorm(x)) in one op: x [B, C, H, W] channels_last or [B, C, T, H, W] channels_last_3d in fp32, bf16 or fp16, any C that
    `groups` divides (at most 4096) -> the same layout and type; statistics and arithmetic in fp32, rounded once.  weight, bias [C] (fp32 or
    x's type, nullable); activation: "none", "relu", "silu", "gelu" (erf form).  Differentiable in x, weight and bias; the backward
    pass keeps x and the statistics only."""
    if x.dim() not in (4, 5):
        raise ValueError(f"group_norm_act: x must be [B, C, H, W] or [B, C, T, H, W], got {tuple(x.shape)}")
    C = x.shape[1]
    if activation not in ACTIVATIONS:
        raise ValueError(f"group_norm_act: activation {activation!r}, takes one of {sorted(ACTIVATIONS)}")
    if x.dtype not in _lib.FLOAT_TYPES:
        raise TypeError(f"group_norm_act: x is {x.dtype}, takes float32, bfloat16 or float16")
    if groups < 1 or C < 1 or C % groups or C > MAX_CHANNELS:
        raise ValueError(f"group_norm_act: {C} channels in {groups} groups (the groups divide the channels, at most {MAX_CHANNELS})")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"group_norm_act: eps {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            if tuple(p.shape) != (C,):
                raise ValueError(f"group_norm_act: {name} must be [{C}], got {tuple(p.shape)}")
            if p.dtype not in (torch.float32, x.dtype):
                raise TypeError(f"group_norm_act: {name} is {p.dtype}, takes float32 or x's type {x.dtype}")
            if p.device != x.device:
                raise ValueError(f"group_norm_act: {name} is on {p.device}, x on {x.device}")
    if not x.is_contiguous(memory_format=_channels_last(x)):
        raise ValueError("group_norm_act: x must be channels-last (x.contiguous(memory_format=torch.channels_last), _3d for five dimensions)")
    if x.shape[2:].numel() > 1 << 30:
        raise ValueError("group_norm_act: more than 2^30 places in a map")
    if x.shape[0] > _lib.MAX_SIZE:
        raise ValueError(f"group_norm_act: {x.shape[0]} maps")
    if not x.is_cuda:
        raise RuntimeError("combo_avs_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback")
    how = (int(groups), float(eps), ACTIVATIONS[activation])
    if _lib.recorded(x, weight, bias):
        return _lib.record(_GroupNormAct, x, weight, bias, *how)
    return _act_forward(x, _param(weight), _param(bias), *how)[0]
