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


CU = [0, 90, 150]


def _calls():
    from native_sparse_attention_triton_b200 import ops

    cu = torch.tensor(CU, dtype=torch.int32).cuda()
    q, k, v = (_rows(150, h, 64, i) for i, h in enumerate((4, 2, 2)))
    wide = [_rows(150, h, 128, i) for i, h in enumerate((4, 2, 2))]
    idx = torch.full((2, 150, 2), -1, dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(90), torch.arange(60)]).cuda()
    idx[:, :, 0] = (pos // 64).int()  # a query's own block
    w = torch.randn(2, 32 * 64, 64, device="cuda").to(BF) * 0.02
    gate = torch.rand(150, 4, 3, device="cuda").to(BF)
    freq = torch.rand(32, device="cuda")
    return {
        "sliding_window_attention": (wide, lambda a, b, c: ops.sliding_window_attention(a, b, c, cu, 90, 20)),
        "flash_attention_varlen": ([q, k, v], lambda a, b, c: ops.flash_attention_varlen(a, b, c, cu, cu, 90, 90, True)),
        "sink_window_attention": ([q, k, v], lambda a, b, c: ops.sink_window_attention(a, b, c, cu, 20, 2)),
        "topk_sparse_attention": ([q, k, v], lambda a, b, c: ops.topk_sparse_attention(a, b, c, idx, 64, cu)),
        "gate_combine": ([gate, q, q.clone(), q.clone()], ops.gate_combine),
        "rope": ([q], lambda a: ops.rope(a, freq, cu)),
        "linear_compress": ([k, w], lambda a, b: ops.linear_compress(a, b, cu, 32, 16)[0]),
    }


@pytest.mark.parametrize("name", ["sliding_window_attention", "flash_attention_varlen", "sink_window_attention", "topk_sparse_attention", "gate_combine",
                                  "rope", "linear_compress"])
def test_leaves_that_a_living_graph_holds(name):
    """Refused before the engine would have the default stream wait for the one that is captured; captured once that graph is gone."""
    from native_sparse_attention_triton_b200 import device_status

    leaves, call = _calls()[name]
    leaves = [x.requires_grad_(True) for x in leaves]
    alive = call(*leaves)
    do = torch.ones_like(alive)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad([call(*leaves)], leaves, [do])
    torch.cuda.synchronize()
    want = torch.autograd.grad([alive], leaves, [do])
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad([call(*leaves)], leaves, [do])
    graph.replay()
    for a, b in zip(want, grads):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=1e-3)
    assert device_status() == 0
