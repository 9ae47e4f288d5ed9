"""Infinities in one element of q, k, v or of the output's gradient: outputs and gradients have the infinities and NaN of the definition, summed in 64
bits over the pairs that the mask lets through and no others."""
import math

import pytest
import torch

from tests.sink_paged_refs import assert_within, sink_window, window_mask
from tests.test_gpu_sink_window import _cu, _inputs

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
INF = float("inf")


def _definition(q, k, v, do, window, sinks):
    """[o, dq, dk, dv] in 64 bits; a sum over d or over pairs has the terms that are there, so that 0 times infinity of a hidden pair is not among them."""
    n, hq, d = q.shape
    g, scale = hq // k.shape[1], 1 / math.sqrt(d)
    see = window_mask(n, window, sinks, q.device)
    out = [torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in (q, q, k, v)]
    for h in range(hq):
        qh, kh, vh, gh = (x.double() for x in (q[:, h], k[:, h // g], v[:, h // g], do[:, h]))
        for i in range(n):
            j = see[i].nonzero()[:, 0]
            p = torch.softmax((kh[j] * qh[i]).sum(1) * scale, 0)
            o = (p[:, None] * vh[j]).sum(0)
            ds = p * ((vh[j] * gh[i]).sum(1) - (o * gh[i]).sum()) * scale
            out[0][i, h] = o
            out[1][i, h] = (ds[:, None] * kh[j]).sum(0)
            out[2][j, h // g] += ds[:, None] * qh[i]
            out[3][j, h // g] += p[:, None] * gh[i]
    return out


@pytest.mark.parametrize("hq,hkv,d,dtype", [(2, 2, 128, BF), (4, 2, 64, FP), (4, 1, 128, BF), (4, 1, 64, BF)])
@pytest.mark.parametrize("bad", [INF, -INF])
@pytest.mark.parametrize("which,at", [(w, a) for w in range(4) for a in (1, 139, 148)])
def test_one_infinite_element(hq, hkv, d, dtype, bad, which, at):
    from native_sparse_attention_triton_b200 import device_status, ops

    n, window, sinks = 150, 40, 3
    x = list(_inputs([n], hq, hkv, d, dtype, seed=12))
    _, bound = sink_window(*x[:3], [n], window, sinks, x[3])
    x[which][at, x[which].shape[1] - 1, 17] = bad
    want = _definition(*x, window, sinks)
    leaves = [t.requires_grad_(True) for t in x[:3]]
    o = ops.sink_window_attention(*leaves, _cu([n]), window, sinks)
    got = (o.detach(), *torch.autograd.grad([o], leaves, [x[3]]))
    for name, y, w, t in zip(("o", "dq", "dk", "dv"), got, want, bound):
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            off = kind(y) != kind(w)
            assert not off.any(), f"{name}: {kind.__name__} differs at {int(off.sum())} of {off.numel()}, first {off.nonzero()[0].tolist()}"
        # (bounds of the finite inputs hold where nothing depends on the bad one; rows with a probability of zero instead of one of theirs differ)
        same = w.isfinite().all(-1) & (which in (2, 3))
        assert_within(y[same], w[same], t[same], name)
    assert device_status() == 0


@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 1)])
def test_gradients_by_a_probability_far_below_the_smallest_float(hq, hkv):
    """An infinite gradient of an output reaches the value of every key that its query sees, and an infinite value the query's gradient."""
    from native_sparse_attention_triton_b200 import ops

    n, scale = 300, 3.0 / math.sqrt(128)
    q, k, v, do = _inputs([n], hq, hkv, 128, BF, seed=9)
    k[5] = -q[200, ::hq // hkv]  # a logit of about -130 for a query head of each group
    do[200, 0, 7] = INF
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = ops.sink_window_attention(*leaves, _cu([n]), 250, 1, scale)
    dv, = torch.autograd.grad([o], [leaves[2]], [do])
    p = torch.softmax(q.detach()[200, 0].double() @ k.detach()[:201, 0].double().T * scale, 0)
    assert 0 < p[5] < 1e-50
    assert dv[:201, 0, 7].isposinf().all() and dv[5, :, :7].isfinite().all() and dv[201:].isfinite().all()
