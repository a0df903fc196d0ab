"""CPU: what the entry points of group norm with an activation and rotary positions refuse, before anything is launched."""
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
                lambda: group_norm_act(x[:, :4], 2), lambda: group_norm_act(torch.zeros(1, 4100, 1, 1), 2)):
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
    assert lib.combo_groupnorm_act_workspace(2, 9, 8, 2, 0, 0) == 8 and lib.combo_groupnorm_act_workspace(2, 9, 8, 2, 0, 1) == 40
    assert lib.combo_groupnorm_act_forward(one, 0, 0, 1, 9, 8, 3, 1e-5, 0, 0, one, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_forward(one, 0, 0, 1, 9, 8, 2, 1e-5, 4, 0, one, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_forward(one + 2, 0, 0, 1, 9, 8, 2, 1e-5, 0, 0, one, one, one, one, 0) == 1
    assert lib.combo_groupnorm_act_backward(0, one, 0, 0, one, one, 1, 9, 8, 2, 0, 0, one, one, 0, 0, 0) == 1
