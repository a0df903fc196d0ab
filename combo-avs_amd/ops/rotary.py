"""Rotary positions over several axes on csrc/rotary.hip: queries and keys of video or image tokens are turned by their (frame, row,
column) coordinates, in place of the additive sine encoding the reference's decoder uses (position_encoding.py:29-48)."""
import ctypes
import functools
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib

_POS_TYPES = {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3}
MAX_HEAD_DIM, MAX_AXES = 256, 8


@functools.lru_cache(maxsize=256)
def _tables(sections, base, shared_ladder):
    """-> (sections as a C array, turns per unit of position of every pair as a C array)"""
    total, turns, done = sum(sections), [], 0
    for n in sections:
        for i in range(n):
            turns.append(base ** -((done + i) / total if shared_ladder else i / n) / (2 * math.pi))
        done += n
    return (ctypes.c_int * len(sections))(*sections), (ctypes.c_double * max(1, total))(*turns)


def _rotate(x, positions, sections, base, interleaved, shared_ladder, inverse):
    B, N, H, D = x.shape
    y = torch.empty((B, N, H, D), device=x.device, dtype=x.dtype)
    if y.numel() == 0:
        return y
    if x.stride(3) != 1 or (interleaved and any(s % 2 for s in x.stride()[:3])) or (interleaved and x.data_ptr() % (2 * x.element_size())):
        x = x.clone(memory_format=torch.contiguous_format)  # the kernel reads whole pairs of a contiguous last dimension
    sec, turns = _tables(sections, base, shared_ladder)
    pb = positions.stride(0) if positions.dim() == 3 else 0
    with _lib.device_of(x) as stream:
        _lib.check(_lib.lib().combo_rotary_axes(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2), _lib.FLOAT_TYPES[x.dtype],
                                                positions.data_ptr(), _POS_TYPES[positions.dtype], pb, positions.stride(-2),
                                                positions.stride(-1), B, N, H, D, len(sections), sec, turns, 1 if interleaved else 0,
                                                1 if inverse else 0, y.data_ptr(), stream), "combo_rotary_axes")
    return y


class _Rotary(Function):
    @staticmethod
    def forward(ctx, x, positions, how):
        ctx.save_for_backward(positions)
        ctx.how = how
        return _rotate(x, positions, *how, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (positions,) = ctx.saved_tensors
        return _rotate(dy, positions, *ctx.how, True), None, None


def rotary_axes(x, positions, sections, base=10000.0, interleaved=False, shared_ladder=False):
    """x [B, N, H, D] (fp32 / bf16 / fp16, any strides) with the first 2 * sum(sections) values of every head turned by the token's
    positions; the values behind them pass through.  -> contiguous [B, N, H, D] of x's type, differentiable in x.

    positions [N, A] or [B, N, A] (fp32 / fp64 / int32 / int64, any strides; no gradient): one coordinate per axis.  sections: the
    number of pairs of each of the A axes, in order.  Pair i of an axis with n pairs turns by position * base ** (-i / n) (every axis
    has its own ladder of frequencies); shared_ladder: pair j of all P turns by its axis' position * base ** (-j / P).  With
    P = sum(sections), pair j is the values (j, j + P), or (2 j, 2 j + 1) when interleaved.  Angles are formed in 64 bits."""
    if x.dim() != 4:
        raise ValueError(f"rotary_axes: x must be [B, N, H, D], got {tuple(x.shape)}")
    if x.dtype not in _lib.FLOAT_TYPES:
        raise TypeError(f"rotary_axes: x is {x.dtype}, takes float32, bfloat16 or float16")
    if positions.dtype not in _POS_TYPES:
        raise TypeError(f"rotary_axes: positions are {positions.dtype}, takes float32, float64, int32 or int64")
    sections = tuple(int(n) for n in sections)
    B, N, _, D = x.shape
    if positions.device != x.device:
        raise ValueError("rotary_axes: x and positions are on different devices")
    if tuple(positions.shape) not in ((N, len(sections)), (B, N, len(sections))):
        raise ValueError(f"rotary_axes: positions must be [{N}, {len(sections)}] or [{B}, {N}, {len(sections)}], got {tuple(positions.shape)}")
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or 2 * sum(sections) > D:
        raise ValueError(f"rotary_axes: sections {sections}: 1 to {MAX_AXES} axes, not negative, at most half of the head dimension {D}")
    if D % 2 or D > MAX_HEAD_DIM:
        raise ValueError(f"rotary_axes: head dimension {D}: even, at most {MAX_HEAD_DIM}")
    if max(x.shape) > _lib.MAX_SIZE:
        raise ValueError(f"rotary_axes: sizes beyond 2^31: {tuple(x.shape)}")
    base = float(base)
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"rotary_axes: base {base}")
    if positions.requires_grad and torch.is_grad_enabled():
        raise ValueError("rotary_axes: positions have no gradient here; detach them")
    if not (x.is_cuda and positions.is_cuda):
        raise RuntimeError("combo_avs_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback")
    how = (sections, base, bool(interleaved), bool(shared_ladder))
    if _lib.recorded(x, positions):
        return _lib.record(_Rotary, x, positions, how)
    return _rotate(x, positions, *how, False)


def grid_positions(*sizes, device=None, dtype=torch.float32):
    """Coordinates of the tokens of a grid, last axis fastest: grid_positions(T, H, W) -> [T * H * W, 3]."""
    axes = [torch.arange(n, device=device, dtype=dtype) for n in sizes]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, len(sizes))
