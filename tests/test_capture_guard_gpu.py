"""An eager autograd graph that lives on the default stream while a backward pass of the same leaves is captured: the captured backward pass
would have to join the default stream, which ends the process; the ops refuse the capture, and take it once the graph is gone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    from combo_avs_amd.ops.cross_attention import cross_attention
    from combo_avs_amd.ops.groupnorm import group_norm_act
    from combo_avs_amd.ops.rotary import rotary_axes
    x = torch.randn(2, 40, 4, 16, device="cuda").bfloat16().requires_grad_(True)
    m = torch.randn(2, 8, 6, 6, device="cuda").contiguous(memory_format=torch.channels_last)
    w = torch.ones(8, device="cuda", requires_grad=True)
    k = torch.randn(2, 40, 4, 16, device="cuda").bfloat16()
    pos = torch.rand(40, 1, device="cuda")
    return {"cross": (lambda: cross_attention(x, k, k), x), "norm": (lambda: group_norm_act(m, 2, w), w), "rotary": (lambda: rotary_axes(x, pos, (4,)), x)}


@pytest.mark.parametrize("name", ["cross", "norm", "rotary"])
def test_capture_beside_a_living_eager_graph_is_refused(name):
    call, leaf = ops()[name]
    want = torch.autograd.grad(call().float().sum(), leaf)[0]
    alive = call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            call()
    assert alive.requires_grad
    del alive, graph
    side = torch.cuda.Stream()  # a graph recorded on another stream may live on
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(call().float().sum(), leaf)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_capture_is_refused_for_norm_parameters_of_the_maps_type():
    """parameters that the op widens for itself are leaves too"""
    from combo_avs_amd.ops.groupnorm import group_norm_act
    m = torch.randn(2, 8, 6, 6, device="cuda").bfloat16().contiguous(memory_format=torch.channels_last)
    w, b = (torch.rand(8, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
    alive = group_norm_act(m, 2, w, b, activation="silu")
    dw, db = torch.autograd.grad(alive, (w, b), torch.ones_like(alive), retain_graph=True)
    w32, b32 = (t.detach().float().requires_grad_(True) for t in (w, b))
    dw32, db32 = torch.autograd.grad(group_norm_act(m, 2, w32, b32, activation="silu"), (w32, b32), torch.ones_like(alive))
    assert torch.equal(dw, dw32.bfloat16()) and torch.equal(db, db32.bfloat16())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            group_norm_act(m, 2, w, b, activation="silu")
