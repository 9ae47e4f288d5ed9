"""Backward passes captured in a CUDA graph while a graph of the default stream that holds the same leaves lives."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _rows(n, h, d, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, h, d, generator=g, device="cuda").to(BF)


@pytest.mark.parametrize("asked,held", [((0,), (1, 2)), ((1,), (0,)), ((1, 2), (0,)), ((0, 2), (1,))])
def test_graphs_of_inputs_that_nobody_asks_about(asked, held):
    """The engine hands over the gradients that are asked for; what another graph holds besides does not matter."""
    from native_sparse_attention_triton_b200 import device_status, ops

    cu = torch.tensor([0, 90, 150], dtype=torch.int32).cuda()
    x, do = [_rows(150, h, 64, i).requires_grad_(True) for i, h in enumerate((4, 2, 2))], _rows(150, 4, 64, 3)
    alive = ops.sink_window_attention(*[t if i in held else t.detach() for i, t in enumerate(x)], cu, 10, 2)
    leaves = [x[i] for i in asked]

    def step():
        return torch.autograd.grad([ops.sink_window_attention(*x, cu, 10, 2)], leaves, [do])

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    graph.replay()
    for a, b in zip(grads, step()):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=1e-5)
    assert device_status() == 0 and alive.shape == x[0].shape
