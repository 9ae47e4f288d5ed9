"""sink_window_attention against its definition in 64 bits, forward and backward, within the bounds its roundings give."""
import pytest
import torch

from tests.sink_paged_refs import SLACK, assert_within, half_step, least_step, sink_window, window_mask

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _cu(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()


def _inputs(lens, hq, hkv, d, dtype, seed=0, extra=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(lens) + extra
    mk = lambda h, s=1.0: (torch.randn(n, h, d, generator=g, device="cuda") * s).to(dtype)
    return mk(hq, 2.0), mk(hkv), mk(hkv), mk(hq)


def _check(lens, hq, hkv, d, dtype, window, sinks, seed=0, scale=None):
    from native_sparse_attention_triton_b200 import device_status, ops

    q, k, v, do = _inputs(lens, hq, hkv, d, dtype, seed)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o = ops.sink_window_attention(q, k, v, _cu(lens), window, sinks, scale)
    grads = torch.autograd.grad([o], leaves, [do])
    value, bound = sink_window(q.detach(), k.detach(), v.detach(), lens, window, sinks, do, scale)
    for name, got, x, t in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), value, bound):
        assert got.dtype == dtype
        assert_within(got, x, t, name)
    assert device_status() == 0


LENGTHS = [
    ([1], 0, 0), ([1], 5, 3), ([2], 0, 1), ([1, 1, 3], 1, 1), ([0, 5, 0, 130, 0], 16, 2), ([127, 128, 129], 128, 4), ([300], 0, 0), ([300], 0, 1),
    ([700], 63, 8), ([513], 512, 4), ([515, 77], 127, 16), ([900], 100, 7), ([640, 3], 10 ** 9, 2), ([260], 32, 10 ** 9), ([1100], 64, 128),
    ([1100], 200, 130), ([600], 17, 255), ([1000, 1, 333], 256, 64), ([1025], 1, 9),
]


@pytest.mark.parametrize("lens,window,sinks", LENGTHS)
def test_lengths_windows_and_sinks(lens, window, sinks):
    _check(lens, 16, 2, 128, BF, window, sinks)


@pytest.mark.parametrize("lens,window,sinks", LENGTHS[4::3])
def test_lengths_windows_and_sinks_head_dim_64_fp16(lens, window, sinks):
    _check(lens, 8, 2, 64, FP, window, sinks)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (2, 1), (4, 1), (12, 3), (8, 1), (16, 1), (32, 2), (10, 5)])
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, BF), (128, FP)])
def test_head_layouts(hq, hkv, d, dtype):
    _check([431, 66], hq, hkv, d, dtype, 70, 5)


@pytest.mark.parametrize("window", [512, 1500])
def test_longer_than_a_cta(window):
    """Key tiles whose tokens take several CTAs of the backward pass, sinks of several chunks of tokens."""
    _check([5000, 2100], 16, 2, 128, BF, window, 12)


def test_a_scale_of_its_own():
    _check([333], 8, 2, 128, BF, 60, 4, scale=0.3)


def test_many_short_sequences():
    _check([(i * 7) % 19 for i in range(150)], 8, 1, 128, BF, 6, 2)


def test_without_sinks_it_is_the_sliding_window():
    from native_sparse_attention_triton_b200 import ops

    lens = [700, 130]
    q, k, v, _ = _inputs(lens, 16, 2, 128, BF)
    cu = _cu(lens)
    a, b = ops.sink_window_attention(q, k, v, cu, 100, 0), ops.sliding_window_attention(q, k, v, cu, 700, 100)
    value, bound = sink_window(q, k, v, lens, 100, 0)
    assert_within(a, value[0], bound[0])
    assert_within(b, value[0], bound[0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_rows_of_no_sequence_reach_nothing(bad):
    """A padded batch: rows behind the last sequence hold anything; their output and gradients are zero."""
    from native_sparse_attention_triton_b200 import ops

    lens, extra = [130, 77], 200
    q, k, v, do = _inputs(lens, 8, 2, 128, BF, extra=extra)
    n = sum(lens)
    for x in (q, k, v, do):
        x[n:] = bad
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o = ops.sink_window_attention(q, k, v, _cu(lens), 50, 3)
    grads = torch.autograd.grad([o], leaves, [do])
    value, bound = sink_window(q.detach()[:n], k.detach()[:n], v.detach()[:n], lens, 50, 3, do[:n])
    for name, got, x, t in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), value, bound):
        assert_within(got[:n], x, t, name)
        assert (got[n:] == 0).all(), name


@pytest.mark.parametrize("which", range(4))
def test_a_sequence_that_is_not_finite_leaves_its_neighbours_alone(which):
    from native_sparse_attention_triton_b200 import ops

    lens = [61, 90, 45]
    x = list(_inputs(lens, 8, 2, 128, BF))
    clean = [t.clone() for t in x]
    x[which][61:151] = float("nan")
    leaves = [t.requires_grad_(True) for t in x[:3]]
    o = ops.sink_window_attention(*leaves, _cu(lens), 30, 4)
    grads = torch.autograd.grad([o], leaves, [x[3]])
    value, bound = sink_window(*clean[:3], lens, 30, 4, clean[3])
    for got, val, t in zip((o.detach(), *grads), value, bound):
        for part in (slice(0, 61), slice(151, 196)):
            assert_within(got[part], val[part], t[part])


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which,at", [(w, a) for w in range(4) for a in (2, 7, 150, 399)])
def test_a_value_that_is_not_finite_reaches_what_depends_on_it_alone(d, dtype, bad, which, at):
    """One row of q, k, v or of the output's gradient.  What the definition makes depend on it, and nothing else, may differ."""
    from native_sparse_attention_triton_b200 import ops

    n, window, sinks = 400, 60, 5
    x = list(_inputs([n], 8, 2, d, dtype))
    value, bound = sink_window(*x[:3], [n], window, sinks, x[3])
    x[which][at] = bad
    leaves = [t.requires_grad_(True) for t in x[:3]]
    o = ops.sink_window_attention(*leaves, _cu([n]), window, sinks)
    grads = torch.autograd.grad([o], leaves, [x[3]])
    see = window_mask(n, window, sinks, "cuda")  # [query, key]
    queries = see[:, at] if which in (1, 2) else torch.arange(n, device="cuda") == at  # with another output or dq
    keys = (see & queries[:, None]).any(0)  # with another dk or dv
    none = torch.zeros_like(queries)
    touched = [none if which == 3 else queries, queries, keys, keys]
    for name, got, val, t, hit in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), value, bound, touched):
        assert_within(got[~hit], val[~hit], t[~hit], name)


def test_batches_of_nothing_finite_end():
    from native_sparse_attention_triton_b200 import device_status, ops

    q, k, v, do = _inputs([700, 3], 8, 2, 128, BF)
    leaves = [x.requires_grad_(True) for x in (q, k, torch.full_like(v, float("nan")))]
    o = ops.sink_window_attention(*leaves, _cu([700, 3]), 100, 4)
    dq, dk, dv = torch.autograd.grad([o], leaves, [do])
    assert o.isnan().all() and dq.isnan().all() and dk.isnan().all() and dv.isfinite().all()
    assert device_status() == 0


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
def test_strided_inputs_and_gradients(d, dtype):
    """q, k and v as slices of one tensor, an output gradient with heads outermost, rows at odd offsets (copied)."""
    from native_sparse_attention_triton_b200 import ops

    lens = [200, 133]
    n = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(n, 12, d, generator=g, device="cuda").to(dtype)
    odd = torch.randn(n * 2 * d + 3, generator=g, device="cuda").to(dtype)[3:].view(n, 2, d)
    do = torch.randn(8, n, d, generator=g, device="cuda").to(dtype).transpose(0, 1)
    for k, v in ((qkv[:, 8:10], qkv[:, 10:12]), (qkv[:, 8:12:2], odd.clone())):
        leaves = [x.detach().requires_grad_(True) for x in (qkv[:, :8], k, v)]
        o = ops.sink_window_attention(*leaves, _cu(lens), 40, 3)
        grads = torch.autograd.grad([o], leaves, [do])
        value, bound = sink_window(qkv[:, :8], k, v, lens, 40, 3, do)
        for name, got, x, t in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), value, bound):
            assert_within(got, x, t, name)


def test_broadcast_inputs_and_gradients():
    """Keys and values of one head (or one row) for all heads, an output gradient that is one head's: dimensions with a stride of zero."""
    from native_sparse_attention_triton_b200 import ops

    lens = [200, 133]
    q, k, v, do = _inputs(lens, 8, 1, 128, BF, seed=9)
    for wide_k, wide_do in ((k.expand(-1, 4, -1), do[:, :1].expand(-1, 8, -1)), (k[:1].expand(333, 4, -1), do[:1].expand(333, -1, -1))):
        wide_v = v.expand(-1, 4, -1)
        leaves = [x.detach().requires_grad_(True) for x in (q, wide_k, wide_v)]
        o = ops.sink_window_attention(*leaves, _cu(lens), 40, 3)
        grads = torch.autograd.grad([o], leaves, [wide_do])
        value, bound = sink_window(q, wide_k, wide_v, lens, 40, 3, wide_do)
        for name, got, x, t in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), value, bound):
            assert_within(got, x, t, name)


def test_all_keys_are_sinks_of_many_sequences():
    """num_sinks far beyond the lengths: plain causal attention, all of whose key rows are summed up."""
    _check([3, 200, 0, 1, 129, 64], 8, 2, 128, BF, 0, 10 ** 6)
    _check([40] * 30, 4, 4, 64, FP, 3, 200)


def test_a_captured_backward_of_leaves_that_a_living_graph_holds():
    """Refused before the autograd engine would have the default stream wait for the one that is captured."""
    from native_sparse_attention_triton_b200 import device_status, ops

    lens, cu = [100], _cu([100])
    q, k, v, do = _inputs(lens, 4, 2, 64, BF)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    alive = ops.sink_window_attention(*leaves, cu, 10, 2)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            torch.autograd.grad([ops.sink_window_attention(*leaves, cu, 10, 2)], leaves, [do])
    del alive
    torch.cuda.synchronize()
    first = [x.clone() for x in torch.autograd.grad([ops.sink_window_attention(*leaves, cu, 10, 2)], leaves, [do])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad([ops.sink_window_attention(*leaves, cu, 10, 2)], leaves, [do])
    graph.replay()
    for a, b in zip(first, grads):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=1e-5)
    assert device_status() == 0


def test_no_tokens():
    from native_sparse_attention_triton_b200 import ops

    q, k = torch.zeros(0, 4, 128, dtype=BF, device="cuda", requires_grad=True), torch.zeros(0, 2, 128, dtype=BF, device="cuda", requires_grad=True)
    o = ops.sink_window_attention(q, k, k, _cu([0, 0]), 4, 1)
    assert o.shape == q.shape
    o.sum().backward()
    assert q.grad.shape == q.shape and k.grad.shape == k.shape


def test_one_of_the_inputs_differentiated_and_a_second_backward():
    from native_sparse_attention_triton_b200 import ops

    q, k, v, do = _inputs([200], 8, 2, 128, BF)
    k.requires_grad_(True)
    o = ops.sink_window_attention(q, k, v, _cu([200]), 40, 3)
    first, = torch.autograd.grad([o], [k], [do], retain_graph=True)
    second, = torch.autograd.grad([o], [k], [do])
    value, bound = sink_window(q, k.detach(), v, [200], 40, 3, do)
    assert_within(first, value[2], bound[2])
    assert_within(second, value[2], bound[2])
    with pytest.raises(RuntimeError):
        torch.autograd.grad([o], [k], [do])
    with torch.no_grad():
        assert not ops.sink_window_attention(q, k, v, _cu([200]), 40, 3).requires_grad


def test_on_a_stream_of_its_own_and_captured():
    """Forward and backward on a side stream; captured in a CUDA graph and replayed with other inputs in place."""
    from native_sparse_attention_triton_b200 import ops

    lens = [300, 200]
    cu = _cu(lens)
    q, k, v, do = _inputs(lens, 16, 2, 128, BF, seed=1)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        o = ops.sink_window_attention(*leaves, cu, 64, 4)
        return (o.detach(), *torch.autograd.grad([o], leaves, [do]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = step()
    torch.cuda.current_stream().wait_stream(side)
    value, bound = sink_window(q.detach(), k.detach(), v.detach(), lens, 64, 4, do)
    for got, x, t in zip(outs, value, bound):
        assert_within(got, x, t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    other = _inputs(lens, 16, 2, 128, BF, seed=2)
    with torch.no_grad():
        for dst, src in zip((q, k, v, do), other):
            dst.copy_(src)
    graph.replay()
    value, bound = sink_window(*other[:3], lens, 64, 4, other[3])
    for got, x, t in zip(outs, value, bound):
        assert_within(got, x, t)


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, BF), (128, FP), (64, FP)])
@pytest.mark.parametrize("lens,window,sinks", [([9, 1, 2], 3, 1), ([700, 130], 100, 4), ([513], 512, 64)])
def test_an_output_for_a_backward_pass_has_the_probabilities_in_two_parts(d, dtype, lens, window, sinks):
    """Each p = hi + lo is off by at most h * h (lo, at most h of p, is rounded itself), or by the least step of the type; what is left is the
    output's own rounding, h of it, and SLACK.  One part would be off by h of each p."""
    from native_sparse_attention_triton_b200 import ops

    q, k, v, _ = _inputs(lens, 8, 2, d, dtype, seed=3)
    o = ops.sink_window_attention(q.requires_grad_(True), k, v, _cu(lens), window, sinks).detach()
    q, h, u, start = q.detach(), half_step(dtype), least_step(dtype), 0
    for n in lens:
        part = slice(start, start + n)
        see = window_mask(n, window, sinks, "cuda")
        for head in range(8):
            vh = v[part, head // 4].double()
            p = torch.softmax((q[part, head].double() @ k[part, head // 4].double().T * d ** -0.5).masked_fill(~see, -float("inf")), 1)
            x = p @ vh
            assert_within(o[part, head], x, h * x.abs() + u + (h * h + SLACK) * (p @ vh.abs()) + u * (see.double() @ vh.abs()), "o")
        start += n
