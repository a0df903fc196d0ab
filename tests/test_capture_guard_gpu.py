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
