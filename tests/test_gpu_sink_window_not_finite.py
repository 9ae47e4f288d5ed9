"""sink_window_attention on values that are not finite: what depends on them by the definition is not a number, everything else is as it was.

The dK/dV pass has two ways to end: key tiles whose tokens one CTA has write their rows themselves (as many key heads as query heads, or many key
tiles), others are summed up over several CTAs (few key tiles).  Both compute the rows that are not finite one by one."""
import math

import pytest
import torch

from tests.sink_paged_refs import assert_within, sink_window, window_mask
from tests.test_gpu_sink_window import _cu, _inputs

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def _run(x, cu, window, sinks):
    from native_sparse_attention_triton_b200 import device_status, ops

    leaves = [t.requires_grad_(True) for t in x[:3]]
    o = ops.sink_window_attention(*leaves, cu, window, sinks)
    grads = torch.autograd.grad([o], leaves, [x[3]])
    for t in leaves:
        t.requires_grad_(False)
    assert device_status() == 0
    return (o.detach(), *grads)


# 8/8 and 8/4 heads: one CTA has a key tile's tokens; 8/1: two have them
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 8, 128, BF), (8, 4, 64, FP), (8, 1, 128, BF), (8, 1, 64, FP)])
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("at", [2, 127, 150, 383, 399])
def test_a_row_of_nan(hq, hkv, d, dtype, which, at):
    """One row of q, k, v or of the output's gradient, among the sinks, in key tiles of 128 rows and in the last, shorter one."""
    n, window, sinks = 400, 60, 5
    x = list(_inputs([n], hq, hkv, d, dtype, seed=4))
    value, bound = sink_window(*x[:3], [n], window, sinks, x[3])
    x[which][at] = NAN
    got = _run(x, _cu([n]), window, sinks)
    see = window_mask(n, window, sinks, "cuda")  # [query, key]
    here = torch.arange(n, device="cuda") == at
    queries = see[:, at] if which in (1, 2) else here
    keys = (see & queries[:, None]).any(0)
    none = torch.zeros_like(here)
    # v and do do not change the probabilities: with v's row dV stays as it is, with do's row the output does
    touched = [none if which == 3 else queries, queries, keys, none if which == 2 else keys]
    for name, y, val, t, hit in zip(("o", "dq", "dk", "dv"), got, value, bound, touched):
        assert_within(y[~hit], val[~hit], t[~hit], name)
        assert y[hit].isnan().all(), name


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1)])
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
def test_infinities_in_the_values(hq, hkv, d, dtype):
    """A column of V: the outputs that see it have its infinity, forward alone and in front of a backward pass; both signs make no number."""
    from native_sparse_attention_triton_b200 import ops

    n, window, sinks = 500, 90, 3
    q, k, v, do = _inputs([n], hq, hkv, d, dtype, seed=6)
    v[1, :, 5], v[200, :, 5], v[300, :, 9], v[444, :, 9] = INF, -INF, -INF, INF
    see = window_mask(n, window, sinks, "cuda")
    want = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    for h in range(hq):
        p = torch.softmax((q[:, h].double() @ k[:, h * hkv // hq].double().T / math.sqrt(d)).masked_fill(~see, -INF), 1)
        vh = v[:, h * hkv // hq].double()
        want[:, h] = p @ vh.nan_to_num(0, 0, 0)
        for key, col in ((1, 5), (200, 5), (300, 9), (444, 9)):
            want[:, h, col] += torch.where(see[:, key], vh[key, col], 0.0)
    _, bound = sink_window(q, k, v.nan_to_num(0, 0, 0), [n], window, sinks)
    with_graph = _run([q, k, v, do], _cu([n]), window, sinks)[0]
    for o in (with_graph, ops.sink_window_attention(q, k, v, _cu([n]), window, sinks)):
        o = o.double()
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(o), kind(want)), kind.__name__
        fine = want.isfinite()
        assert_within(o[fine], want[fine], bound[0][fine], "o")



@pytest.mark.parametrize("which", [0, 3])
def test_many_key_heads_of_sixteen_queries(which):
    """Groups of 16 at head_dim 128 whose key tiles one CTA has (40 key heads x 8 tiles): every row against the definition, then a row of NaN."""
    n, window, sinks, hq, hkv = 900, 40, 4, 640, 40
    x = list(_inputs([n], hq, hkv, 128, BF, seed=8))
    heads = [0, 17, 39]
    pick = lambda y: [torch.cat([y[0][:, h * 16:h * 16 + 16] for h in heads], 1), *(torch.stack([t[:, h] for h in heads], 1) for t in y[1:3]),
                      torch.cat([y[3][:, h * 16:h * 16 + 16] for h in heads], 1)]
    sub = pick(x)
    value, bound = sink_window(*sub[:3], [n], window, sinks, sub[3])
    for at in (None, 500, 899):
        y = [t.clone() for t in x]
        if at is not None:
            y[which][at] = NAN
        got = _run(y, _cu([n]), window, sinks)
        got = pick([got[1], got[2], got[3], got[0]])  # dq, dk, dv, o
        see = window_mask(n, window, sinks, "cuda")
        here = torch.arange(n, device="cuda") == (-1 if at is None else at)
        keys = (see & here[:, None]).any(0)
        touched = [here, keys, keys, here if which == 0 else torch.zeros_like(here)]
        for name, g, val, t, hit in zip(("dq", "dk", "dv", "o"), got, (*value[1:], value[0]), (*bound[1:], bound[0]), touched):
            assert_within(g[~hit], val[~hit], t[~hit], name)
            assert g[hit].isnan().all(), name


@pytest.mark.parametrize("graph", [False, True])
def test_rows_that_are_all_minus_infinity(graph):
    """0 / 0: a query all of whose logits are minus infinity has no number, like those behind it that see such keys alone."""
    from native_sparse_attention_triton_b200 import device_status, ops

    lens = [1, 70, 200]
    q, k, v, do = _inputs(lens, 4, 2, 128, BF, seed=7)
    q.abs_()
    k[0, 0, 3], k[1:30, 1, 4] = -INF, -INF
    x = [t.requires_grad_(graph) for t in (q, k, v)]
    o = ops.sink_window_attention(*x, _cu(lens), 10, 2).detach()
    want = torch.zeros(271, 4, dtype=torch.bool, device="cuda")
    want[0, :2], want[1:30, 2:] = True, True
    assert torch.equal(o.isnan().all(-1), want) and torch.equal(o.isnan().any(-1), want)
    assert device_status() == 0


@pytest.mark.parametrize("graph", [False, True])
def test_a_value_whose_probability_is_far_below_the_smallest_float(graph):
    """A probability is above zero, however small, so that infinity times it is infinity."""
    from native_sparse_attention_triton_b200 import ops

    n = 300
    q, k, v, _ = _inputs([n], 4, 2, 128, BF, seed=9)
    k[5] = -q[200, ::2]  # logits of about -130 for two heads of query 200
    v[5, :, 7] = INF
    x = [t.requires_grad_(graph) for t in (q, k, v)]
    o = ops.sink_window_attention(*x, _cu([n]), 250, 1, 3.0 / math.sqrt(128)).detach()
    p = torch.softmax(q.detach()[200, 0].double() @ k.detach()[:201, 0].double().T * 3.0 / math.sqrt(128), 0)
    assert 0 < p[5] < 1e-50
    assert o[200, :, 7].isposinf().all() and o[200, :, :7].isfinite().all()
