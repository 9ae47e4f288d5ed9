"""paged_attention_decode on visible rows that hold infinities and NaN: what the definition gives in 64 bits, and nothing else."""
import math

import pytest
import torch

from tests.sink_paged_refs import DECODE_SLACK, assert_within, paged_decode
from tests.test_gpu_paged import Cache

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")
# pairs that lie whole in a warp's run, that several warps of a CTA have parts of, and that several CTAs have
SHAPES = {"whole": [40] * 300, "parts": [300, 33, 1, 70, 500, 64], "ctas": [20000, 5, 3000]}


def _row(c, x, b, j):
    """Row j of sequence b, [heads, d], in place."""
    return x[int(c.table[b, j // c.page]), j % c.page]


def _same_kind(got, want, bound, name):
    """NaN where the definition has NaN, the same infinities, and finite values within their bounds."""
    got, want = got.double(), want.double()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        off = kind(got) != kind(want)
        assert not off.any(), f"{name}: {kind.__name__} differs at {int(off.sum())} of {off.numel()}, first {off.nonzero()[0].tolist()}"
    fine = torch.isfinite(want)
    assert_within(got[fine], want[fine], bound[fine], name)


def _check(c, hq, window=None, sinks=0, weights=False, scale=None, q=None):
    from native_sparse_attention_triton_b200 import device_status, ops

    q = c.queries(hq) if q is None else q
    w = torch.rand(len(c.lens), c.k.shape[2], c.table.shape[1] * c.page, device="cuda") if weights else None
    before = w.clone() if weights else None
    o = ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens, scale, window, sinks, w)
    value, bound, added = paged_decode(q, c.k, c.v, c.table, c.lens, window, sinks, scale)
    _same_kind(o, value, bound, "o")
    if weights:
        for b, (rows, p) in enumerate(added):
            want = before[b].double()
            want[:, rows] += p
            tol = torch.zeros_like(want)
            tol[:, rows] = DECODE_SLACK * p + torch.finfo(torch.float32).eps * want[:, rows]
            _same_kind(w[b], want, tol, f"weights of {b}")
    assert device_status() == 0
    return value


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP), (64, BF), (128, FP)])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_visible_value(shape, bad, d, dtype):
    """A column of one V row of every second sequence."""
    c = Cache(SHAPES[shape], 2, d, 16, dtype)
    for b in range(0, len(c.lens), 2):
        _row(c, c.v, b, (b * 7) % c.lens[b])[b % 2, (b * 5) % d] = bad
    value = _check(c, 16)
    assert (~value.isfinite()).any() and value.isfinite().any()


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("shape", SHAPES)
def test_infinities_of_both_signs(shape, d, dtype):
    """In one column of two rows (NaN, as their sum is), and in a column each of one row."""
    c = Cache(SHAPES[shape], 2, d, 16, dtype)
    for b in range(0, len(c.lens), 2):
        _row(c, c.v, b, 0)[0, 3], _row(c, c.v, b, c.lens[b] - 1)[0, 3] = INF, -INF
        _row(c, c.v, b, c.lens[b] // 2)[1, 9], _row(c, c.v, b, c.lens[b] // 2)[1, 11] = INF, -INF
    _check(c, 8)





def test_a_value_whose_probability_is_far_below_the_smallest_float():
    """A probability is above zero, however small, so that infinity times it is infinity."""
    c = Cache([30, 2000, 20000], 2, 128, 16, BF)
    q = c.queries(8)
    for b, n in enumerate(c.lens):
        _row(c, c.k, b, 0)[:] = (q[b, ::4] * -1).to(BF)  # a logit of about -136 for the first head of a group
        _row(c, c.v, b, 0)[:, 5] = INF
    value = _check(c, 8, scale=3.0 / math.sqrt(128), q=q)
    assert value[:, 0, 5].isposinf().all()


def test_with_a_window_and_sinks():
    c = Cache([5000, 90, 700], 2, 128, 16, BF)
    for b, n in enumerate(c.lens):
        _row(c, c.v, b, 1)[:, 2] = INF       # a sink
        _row(c, c.v, b, n - 20)[:, 7] = NAN  # in the window
    _row(c, c.v, 0, 2000)[:] = NAN           # in neither
    value = _check(c, 8, 100, 4, weights=True)
    assert value[:, :, 2].isposinf().all() and value[:, :, 7].isnan().all() and value[0, 0, 3].isfinite()


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_visible_key_that_is_no_number(shape, d, dtype):
    """Neither the heads that see it nor the sums that they add to have a number."""
    c = Cache(SHAPES[shape], 2, d, 16, dtype)
    for b in range(0, len(c.lens), 2):
        _row(c, c.k, b, (b * 11) % c.lens[b])[1, 6] = NAN
    value = _check(c, 8, weights=True)
    assert value[0, 4:].isnan().all() and value[0, :4].isfinite().all()


@pytest.mark.parametrize("shape", SHAPES)
def test_a_query(shape):
    c = Cache(SHAPES[shape], 2, 128, 16, BF)
    q = c.queries(8)
    q[0, 3, 5], q[-1, 6, 0] = NAN, NAN
    value = _check(c, 8, weights=True, q=q)
    assert value[0, 3].isnan().all() and value[0, 2].isfinite().all()


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_visible_key(shape, bad, d, dtype):
    """Heads whose product with it is minus infinity do not see the row; the others have no number, nor have the sums that they add to."""
    c = Cache(SHAPES[shape], 2, d, 16, dtype)
    for b in range(0, len(c.lens), 2):
        _row(c, c.k, b, (b * 11) % c.lens[b])[1, 6] = bad
    _check(c, 8, weights=True)


@pytest.mark.parametrize("lens", [[1], [40], [700], [9000]])
def test_rows_that_are_all_minus_infinity(lens):
    """0 / 0: the softmax of nothing but minus infinities is no number.  A sequence without rows has zeros."""
    c = Cache(lens + [0, 3], 2, 64, 16, BF)
    q = c.queries(4).abs()
    for j in range(0, lens[0], 16):
        c.k[int(c.table[0, j // 16]), :, 1, 0] = -INF
    value = _check(c, 4, weights=True, q=q)
    assert value[0, 2:].isnan().all() and value[0, :2].isfinite().all() and (value[1] == 0).all()
