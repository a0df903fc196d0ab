"""CPU: what the entry points of group norm with an activation, rotary positions and cross attention refuse, before anything is launched."""
import pytest
import torch


def test_rotary_refusals():
    from combo_avs_amd.ops.rotary import rotary_axes
    x, p = torch.zeros(2, 3, 1, 8), torch.zeros(3, 2)
    for bad in (lambda: rotary_axes(x[0], p, (1, 1)), lambda: rotary_axes(x, p[:2], (1, 1)), lambda: rotary_axes(x, p, (1, 1, 1)),
                lambda: rotary_axes(x, p, (2, 3)), lambda: rotary_axes(x, p, (-1, 2)), lambda: rotary_axes(x, p, (1, 1), base=0.0),
                lambda: rotary_axes(x, p, (1, 1), base=float("nan")), lambda: rotary_axes(x[..., :7], p, (1, 1)),
                lambda: rotary_axes(torch.zeros(2, 3, 1, 258), p, (1, 1)), lambda: rotary_axes(x, torch.zeros(3, 9), (0,) * 9),
                lambda: rotary_axes(x, torch.zeros(3, 0), ()), lambda: rotary_axes(x, p.requires_grad_(True), (1, 1))):
        with pytest.raises(ValueError):
            bad()
    p = p.detach()
    for bad in (lambda: rotary_axes(x.double(), p, (1, 1)), lambda: rotary_axes(x, p.half(), (1, 1)), lambda: rotary_axes(x.long(), p, (1, 1))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="GPU only"):
        rotary_axes(x, p, (1, 1))


def test_group_norm_act_refusals():
    from combo_avs_amd.ops.groupnorm import group_norm_act
    x = torch.zeros(2, 8, 3, 3).contiguous(memory_format=torch.channels_last)
    for bad in (lambda: group_norm_act(x[0], 2), lambda: group_norm_act(x, 3), lambda: group_norm_act(x, 0), lambda: group_norm_act(x, 2, activation="tanh"),
                lambda: group_norm_act(x, 2, torch.ones(7)), lambda: group_norm_act(x, 2, None, torch.ones(8, 1)), lambda: group_norm_act(x.contiguous(), 2),
                lambda: group_norm_act(x[:, :4], 2), lambda: group_norm_act(x, 2, eps=-1e-5), lambda: group_norm_act(x, 2, eps=float("nan")), lambda: group_norm_act(torch.zeros(1, 4100, 1, 1), 2)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: group_norm_act(x.double(), 2), lambda: group_norm_act(x, 2, torch.ones(8).half()), lambda: group_norm_act(x.int(), 2)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="GPU only"):
        group_norm_act(x, 2)


def test_entry_points_refuse_bad_arguments_without_a_launch():
    import ctypes
    from combo_avs_amd import _lib
    lib = _lib.lib()
    one = 4096  # (never dereferenced: every call below is refused on the host)
    sec, turns = (ctypes.c_int * 2)(1, 1), (ctypes.c_double * 2)(0.1, 0.1)

    def rotary(D=8, axes=2, pos_type=0, dtype=0, B=1, x=one, H=1):
        return lib.combo_rotary_axes(x, 8, 8, 8, dtype, one, pos_type, 2, 2, 1, B, 1, H, D, axes, sec, turns, 0, 0, one, 0)
    assert all(rc == 1 for rc in (rotary(D=7), rotary(D=2), rotary(D=258), rotary(axes=0), rotary(axes=9), rotary(pos_type=4), rotary(dtype=3),
                                  rotary(B=0), rotary(x=0), rotary(x=4098), rotary(H=1 << 25)))
    assert lib.combo_groupnorm_act_workspace(1, 9, 8, 3, 0, 0) == -1 and lib.combo_groupnorm_act_workspace(1, 9, 4104, 2, 0, 0) == -1
    assert lib.combo_groupnorm_act_workspace(1, (1 << 30) + 1, 1, 1, 0, 0) == -1 and lib.combo_groupnorm_act_workspace(1, 1 << 30, 1, 1, 0, 0) > 0
    assert lib.combo_groupnorm_act_workspace(1 << 18, 1, 4096, 2, 0, 0) == -1  # more workgroups than a launch holds
    assert lib.combo_groupnorm_act_workspace(2, 9, 8, 2, 0, 0) == 0 and lib.combo_groupnorm_act_workspace(2, 9, 8, 2, 0, 1) == 40
    assert lib.combo_groupnorm_act_workspace(2, 9000, 64, 2, 0, 0) > 0
    assert lib.combo_groupnorm_act_forward(one, 0, 0, 2, 9000, 64, 2, 1e-5, 0, 0, 0, one, one, one, 0) == 1  # two launches need their workspace
    assert lib.combo_groupnorm_act_forward(one, 0, 0, 1, 9, 8, 2, 1e-5, 0, 0, 0, one, 0, one, 0) == 1  # mean without rstd
    assert lib.combo_groupnorm_act_forward(one, 0, 0, 1, 9, 8, 3, 1e-5, 0, 0, one, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_forward(one, 0, 0, 1, 9, 8, 2, 1e-5, 4, 0, one, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_forward(one + 2, 0, 0, 1, 9, 8, 2, 1e-5, 0, 0, one, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_backward(0, one, 0, 0, one, one, 1, 9, 8, 2, 0, 0, one, one, 0, 0, 0) == 1


def test_cross_attention_refusals():
    from combo_avs_amd.ops.cross_attention import cross_attention
    q, k = torch.zeros(2, 3, 4, 16).half(), torch.zeros(2, 5, 2, 16).half()
    n = torch.tensor([1, 2], dtype=torch.int32)
    for bad in (lambda: cross_attention(q[0], k, k), lambda: cross_attention(q, k, k[:, :4]), lambda: cross_attention(q[:1], k, k),
                lambda: cross_attention(q, k[..., :8], k[..., :8]), lambda: cross_attention(q[..., :12], k[..., :12], k[..., :12]),
                lambda: cross_attention(q[:, :, :3], k, k), lambda: cross_attention(q, k[:, :, :0], k[:, :, :0]), lambda: cross_attention(q, k, k, scale=0.0),
                lambda: cross_attention(q, k, k, scale=-1.0), lambda: cross_attention(q, k, k, scale=float("nan")),
                lambda: cross_attention(q, k, k, scale=1e39), lambda: cross_attention(q, k, k, scale=1e-60), lambda: cross_attention(q, k, k, n[:1]),
                lambda: cross_attention(q, k, k, blocked=torch.zeros(2, 1, 3, 4, dtype=torch.bool)),
                lambda: cross_attention(q, k, k, blocked=torch.zeros(3, 5, dtype=torch.bool)),
                lambda: cross_attention(q, k, k, blocked=torch.zeros(2, 2, 3, 5, dtype=torch.bool)),
                lambda: cross_attention(torch.zeros(1, 1, 1, 136).half(), torch.zeros(1, 1, 1, 136).half(), torch.zeros(1, 1, 1, 136).half())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cross_attention(q.float(), k.float(), k.float()), lambda: cross_attention(q, k, k.bfloat16()), lambda: cross_attention(q, k, k, n.short()),
                lambda: cross_attention(q, k, k, blocked=torch.zeros(2, 1, 3, 5, dtype=torch.uint8)),
                lambda: cross_attention(q, k, k, blocked=torch.full((2, 1, 3, 5), torch.finfo(torch.float16).min))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="GPU only"):
        cross_attention(q, k, k, n)


def test_cross_attention_entry_points_refuse_without_a_launch():
    from combo_avs_amd import _lib
    from combo_avs_amd.ops.cross_attention import _DESC
    lib, one = _lib.lib(), 4096

    def desc(q=one, qs=(64, 32, 16), B=1, Lq=2, Lk=3, Hq=2, Hk=1, D=16, dtype=1, scale=0.25):
        return _DESC.pack(q, one, one, *qs, *qs, *qs, 0, 0, 0, 0, 0, B, Lq, Lk, Hq, Hk, D, dtype, scale)
    assert lib.combo_cross_attention_workspace(desc(), 0) == 0 and lib.combo_cross_attention_workspace(desc(), 1) >= 16
    for bad in (desc(q=0), desc(q=one + 2), desc(qs=(64, 32, 12)), desc(qs=(64, -32, 16)), desc(B=0), desc(Lq=0), desc(Lk=0), desc(Hk=3), desc(D=12),
                desc(D=136), desc(dtype=0), desc(dtype=3), desc(scale=0.0), desc(scale=float("inf")), desc(scale=float("nan")), desc(Lq=1 << 30),
                desc(B=1 << 24), desc(B=1 << 30), desc(scale=3e38)):
        assert lib.combo_cross_attention_workspace(bad, 0) == -1
        assert lib.combo_cross_attention_forward(bad, one, 0, one, 0) == 1
        assert lib.combo_cross_attention_backward(bad, one, one, one, one, one, one, one, 0) == 1
    assert lib.combo_cross_attention_forward(desc(), 0, 0, one, 0) == 1 and lib.combo_cross_attention_forward(desc(), one + 8, 0, one, 0) == 1
    assert lib.combo_cross_attention_forward(desc(Lk=1000), one, 0, 0, 0) == 1  # split keys need their workspace
    assert lib.combo_cross_attention_backward(desc(), one, one, one, one, one, one, 0, 0) == 1  # dk without dv
    assert lib.combo_cross_attention_pack(one, 1, 1, 1, 1, 0, 1, 1, 1, one, 0) == 1


def test_entry_points_refuse_misaligned_side_tensors():
    from combo_avs_amd import _lib
    from combo_avs_amd.ops.cross_attention import _DESC
    lib, one = _lib.lib(), 4096  # (never dereferenced: every call below is refused on the host)
    for w, b, ws, mean, rstd in ((one + 2, 0, one, one, one), (0, one + 1, one, one, one), (0, 0, one + 4, one, one), (0, 0, one, one + 2, one), (0, 0, one, one, one + 2)):
        assert lib.combo_groupnorm_act_forward(one, w, b, 2, 9000, 64, 2, 1e-5, 0, 0, ws, mean, rstd, one, 0) == 1
        assert lib.combo_groupnorm_act_backward(one, one, w, b, mean, rstd, 2, 9000, 64, 2, 0, 0, ws, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_backward(one, one, 0, 0, one, one, 2, 9000, 64, 2, 0, 0, one, one, one + 2, one, 0) == 1

    def desc(lengths=0, bits=0, bit_stride=0):
        return _DESC.pack(one, one, one, *(64, 32, 16) * 3, lengths, bits, bit_stride, 0, 0, 1, 2, 3, 2, 1, 16, 1, 0.25)
    for bad in (desc(lengths=one + 2), desc(bits=one + 2), desc(bits=one, bit_stride=-1)):
        assert lib.combo_cross_attention_workspace(bad, 0) == -1
        assert lib.combo_cross_attention_forward(bad, one, 0, one, 0) == 1
    assert lib.combo_cross_attention_forward(desc(), one, one + 2, one, 0) == 1
    assert lib.combo_cross_attention_backward(desc(), one, one + 2, one, one, one, one, one, 0) == 1
