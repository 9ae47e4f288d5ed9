"""Scratch of the paged decode operator's running sums: by the rows that a window reaches into, not by the block table's width."""
import pytest
import torch

from native_sparse_attention_triton_b200 import _lib


def _floats(batch, heads, capacity, window, sinks):
    lib = _lib.lib()
    size = lambda weights: lib.nsa_paged_decode_window_scratch_floats(batch, heads, 128, capacity, weights, window, sinks)
    return size(1) - size(0)


def test_a_window_bounds_it():
    for capacity in (4096, 131072, 1 << 30):
        # rows of at most 32 + 1 tiles of a window of 1023 and the key itself, and one of sinks; a log-sum-exp a head; 64 for alignment
        assert _floats(7, 64, capacity, 1023, 4) == 7 * 64 * (34 * 32 + 1) + 64
    assert _floats(7, 64, 512, 1023, 4) == 7 * 64 * (512 + 1) + 64
    assert _floats(1, 1, 40, 0, 0) == 64 + 64 + 1
    assert _floats(3, 8, 1000, 2 ** 30 - 1, 2 ** 30 - 1) == _floats(3, 8, 1000, -1, 0) == 3 * 8 * (1024 + 1) + 64


def test_the_size_without_a_window_is_enough_for_any():
    lib = _lib.lib()
    for window, sinks in [(-1, 0), (0, 0), (31, 1), (100, 33), (10 ** 9, 10 ** 9)]:
        for capacity in (1, 31, 32, 33, 1000, 131072):
            assert lib.nsa_paged_decode_scratch_floats(5, 16, 64, capacity, 1) >= lib.nsa_paged_decode_window_scratch_floats(5, 16, 64, capacity, 1, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,most", [(1023, 4, 40 << 20), (None, 0, 300 << 20)])
def test_memory_of_a_wide_table(window, sinks, most):
    """16 sequences of a table with room for 131 072 rows: with a window little is asked for, without one 268 MB, and nothing of that is kept."""
    from native_sparse_attention_triton_b200 import device_status, ops
    from tests.sink_paged_refs import DECODE_SLACK, assert_within, paged_decode
    from tests.test_gpu_paged import Cache

    c = Cache([2000 + 100 * i for i in range(16)], 2, 128, 64, torch.bfloat16, columns=2048)
    q = c.queries(32)
    w = torch.zeros(16, 2, 131072, device="cuda")
    ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens, None, window, sinks)  # the kept part of the scratch
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for turn in range(3):
        o = ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens, None, window, sinks, w)
        torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < most
    assert torch.cuda.memory_allocated() - before <= (64 << 20) + 2 * o.numel() * 2
    if window is None:
        assert torch.cuda.memory_allocated() - before <= 4 * o.numel()
    value, bound, added = paged_decode(q, c.k, c.v, c.table, c.lens, window, sinks)
    assert_within(o, value, bound)
    for b, (rows, p) in enumerate(added):
        want = torch.zeros(2, 131072, dtype=torch.float64, device="cuda")
        want[:, rows] = 3 * p
        assert ((w[b].double() - want).abs() <= DECODE_SLACK * want + 3 * torch.finfo(torch.float32).eps * want).all()
    assert device_status() == 0
