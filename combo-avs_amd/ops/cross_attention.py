"""Cross attention of queries to encoder states of another length on csrc/cross_attention.hip: bf16 / fp16 with fp32 accumulation, head
dimensions up to 128, grouped heads, a length per sample and a mask.  ops/attention.py is the decoder's own fp32 core at head dimension 32
(transformer_decoder/transformer_decoder.py:99-118); this one serves what it does not take."""
import struct

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib

MAX_HEAD_DIM = 128
_DESC = struct.Struct("3Q9q2Q3q7if")  # combo_cross_attention_t


def _strides(t):
    a, b, c, _ = t.stride()
    l, m, n, _ = t.shape
    return a if l > 1 else 0, b if m > 1 else 0, c if n > 1 else 0


def _readable(t):
    """t as the kernels read it - whole 16-byte vectors of a contiguous last dimension, tokens at most 2^22 elements apart -, copied only where it
    is not laid out so"""
    b, n, h = _strides(t)
    if t.stride(3) == 1 and not (b | n | h) % 8 and n <= 1 << 22 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _packed_bits(blocked, stream):
    """-> (bits [b, h, n, words], strides of a (batch, head, query) in words, 0 where shared)"""
    dims = [n if s else min(n, 1) for n, s in zip(blocked.shape[:3], blocked.stride())]  # (an expanded dimension is packed once)
    Lk = blocked.shape[3]
    words = (Lk + 31) // 32
    bits = torch.empty(dims + [words], device=blocked.device, dtype=torch.int32)
    _lib.check(_lib.lib().combo_cross_attention_pack(blocked.data_ptr(), *blocked.stride(), *dims, Lk, bits.data_ptr(), stream),
               "combo_cross_attention_pack")
    return bits, tuple(s if n > 1 else 0 for s, n in zip(bits.stride(), dims))


def _describe(q, k, v, lengths, bits, bit_strides, scale):
    return _DESC.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q), *_strides(k), *_strides(v), _lib.ptr(lengths), _lib.ptr(bits),
                      *bit_strides, q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], _lib.FLOAT_TYPES[q.dtype], scale)


def _workspace(desc, backward, like):
    n = _lib.lib().combo_cross_attention_workspace(desc, backward)
    if n < 0:
        raise ValueError(f"cross_attention: sizes the kernels do not take: q {tuple(like.shape)}")
    return torch.empty(n, device=like.device, dtype=torch.uint8) if n else None


def _forward(q, k, v, lengths, blocked, scale, keep):
    """-> (out, what the backward pass needs or None)"""
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    q, k, v = _readable(q), _readable(k), _readable(v)
    with _lib.device_of(q) as stream:
        bits, bit_strides = _packed_bits(blocked, stream) if blocked is not None else (None, (0, 0, 0))
        desc = _describe(q, k, v, lengths, bits, bit_strides, scale)
        lse = torch.empty(q.shape[0] * q.shape[1] * q.shape[2], device=q.device, dtype=torch.float32) if keep else None
        ws = _workspace(desc, 0, q)
        _lib.check(_lib.lib().combo_cross_attention_forward(desc, out.data_ptr(), _lib.ptr(lse), _lib.ptr(ws), stream),
                   "combo_cross_attention_forward")
    return out, (q, k, v, lengths, bits, out, lse) if keep else None, bit_strides


class _CrossAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, blocked, scale):
        ctx.scale, ctx.shapes = scale, (q.shape, k.shape)
        ctx.empty = q.numel() == 0 or k.numel() == 0
        if ctx.empty:
            return torch.zeros(q.shape, device=q.device, dtype=q.dtype)
        out, saved, ctx.bit_strides = _forward(q, k, v, lengths, blocked, scale, True)
        ctx.save_for_backward(*saved)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        new = torch.zeros if ctx.empty else torch.empty
        dq = new(ctx.shapes[0], device=dout.device, dtype=dout.dtype)
        want_kv = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]  # (frozen encoder states: their pass is left out)
        dk, dv = (new(ctx.shapes[1], device=dout.device, dtype=dout.dtype) if want_kv else None for _ in range(2))
        if not ctx.empty:
            q, k, v, lengths, bits, out, lse = ctx.saved_tensors
            dout = dout.contiguous()
            if dout.data_ptr() % 16:
                dout = dout.clone()
            with _lib.device_of(q) as stream:
                desc = _describe(q, k, v, lengths, bits, ctx.bit_strides, ctx.scale)
                ws = _workspace(desc, 1, q)
                _lib.check(_lib.lib().combo_cross_attention_backward(desc, out.data_ptr(), lse.data_ptr(), dout.data_ptr(), ws.data_ptr(),
                                                                     dq.data_ptr(), _lib.ptr(dk), _lib.ptr(dv), stream),
                           "combo_cross_attention_backward")
        return dq, dk, dv, None, None, None


def cross_attention(q, k, v, kv_lengths=None, blocked=None, scale=None):
    """softmax(scale q k^T) v over the open keys: q [B, Lq, Hq, D], k / v [B, Lk, Hk, D] (bf16 or fp16, any strides; D a multiple of 8 up to
    128; Hk divides Hq: query head h reads key head h // (Hq // Hk)) -> contiguous [B, Lq, Hq, D], differentiable in q, k and v.

    kv_lengths [B] (int32 / int64, on the GPU): sample b has its first kv_lengths[b] states, clamped to 0 .. Lk.  blocked: bool,
    broadcastable to [B, Hq, Lq, Lk], True = this query does not see this key.  A query that sees no key gets zeros and passes no
    gradient.  States behind a sample's length, and states that a mask shared by all queries and heads blocks, may hold anything; a state
    that only some queries are kept from has to be finite.  scale: positive, D ** -0.5 by default.  Probabilities enter the
    second product in the tensors' type (in two pieces where few rows make the matrix work cheap), as do the score gradients in the
    backward pass, in fp16 at a scale per query and per key that keeps their digits for upstream gradients of any size; sums, statistics and
    gradients accumulate in fp32 in a fixed order (runs repeat bit for bit)."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"cross_attention: q [B, Lq, Hq, D], k and v [B, Lk, Hk, D]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1:3]
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"cross_attention: q, k, v are {q.dtype}, {k.dtype}, {v.dtype}: takes bfloat16 or float16, all three alike")
    if D < 8 or D % 8 or D > MAX_HEAD_DIM:
        raise ValueError(f"cross_attention: head dimension {D}: a multiple of 8, at most {MAX_HEAD_DIM}")
    if Hk < 1 or Hq % Hk:
        raise ValueError(f"cross_attention: {Hq} query heads on {Hk} key heads")
    if max(*q.shape, *k.shape) > _lib.MAX_SIZE:
        raise ValueError(f"cross_attention: sizes beyond 2^31: q {tuple(q.shape)}, k {tuple(k.shape)}")
    scale = float(D ** -0.5 if scale is None else scale)
    if not 1e-37 < scale < 2e38:
        raise ValueError(f"cross_attention: scale {scale}: positive and finite in fp32")
    if kv_lengths is not None:
        if kv_lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"cross_attention: kv_lengths are {kv_lengths.dtype}, takes int32 or int64")
        if tuple(kv_lengths.shape) != (B,):
            raise ValueError(f"cross_attention: kv_lengths must be [{B}], got {tuple(kv_lengths.shape)}")
    if blocked is not None:
        if blocked.dtype != torch.bool:
            raise TypeError(f"cross_attention: blocked is {blocked.dtype}, takes bool (True = not seen)")
        if blocked.dim() != 4 or blocked.shape[3] != Lk or any(n not in (1, full) for n, full in zip(blocked.shape, (B, Hq, Lq))):
            raise ValueError(f"cross_attention: blocked must be broadcastable to [{B}, {Hq}, {Lq}, {Lk}], got {tuple(blocked.shape)}")
    for t in (q, k, v, kv_lengths, blocked):
        if t is not None and not t.is_cuda:
            raise RuntimeError("combo_avs_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback")
        if t is not None and t.device != q.device:
            raise ValueError("cross_attention: the tensors are on different devices")
    if kv_lengths is not None:
        if kv_lengths.dtype == torch.int64:
            kv_lengths = kv_lengths.clamp(0, Lk).to(torch.int32)
        kv_lengths = kv_lengths.contiguous()
    if _lib.recorded(q, k, v):
        return _lib.record(_CrossAttention, q, k, v, kv_lengths, blocked, scale)
    if q.numel() == 0 or k.numel() == 0:
        return torch.zeros(q.shape, device=q.device, dtype=q.dtype)
    return _forward(q, k, v, kv_lengths, blocked, scale, False)[0]
