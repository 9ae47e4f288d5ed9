"""paged_kv_append of rows that are the cache's own: they are taken as they were before the call."""
import pytest
import torch

from tests.test_gpu_paged import BF, Cache, _ints

pytestmark = pytest.mark.gpu


def test_rows_of_the_cache_moved_along():
    """Every row of a page is written one slot further on, in one call: a copy that read what it has written would repeat the first."""
    from native_sparse_attention_triton_b200 import device_status, ops

    n, page = 2000, 2048
    c = Cache([1], 4, 128, page, BF, rows=[page], spare=2)
    at = int(c.table[0, 0])
    for turn in range(5):
        k0, v0 = c.k.clone(), c.v.clone()
        after = ops.paged_kv_append(c.k, c.v, c.table, _ints([1]), c.k[at, :n], c.v[at, :n], _ints([0, n]))
        assert after.tolist() == [n + 1]
        k0[at, 1:n + 1], v0[at, 1:n + 1] = k0[at, :n].clone(), v0[at, :n].clone()
        assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
    # keys from the values' pages and the other way round
    k0, v0 = c.k.clone(), c.v.clone()
    ops.paged_kv_append(c.k, c.v, c.table, _ints([10]), c.v[at, :n], c.k[at, :n], _ints([0, n]))
    k1, v1 = k0.clone(), v0.clone()
    k1[at, 10:n + 10], v1[at, 10:n + 10] = v0[at, :n], k0[at, :n]
    assert torch.equal(c.k, k1) and torch.equal(c.v, v1)
    assert device_status() == 0


def test_rows_beside_the_cache_in_one_storage():
    """Pages and rows cut from one buffer: nothing is copied where they do not meet."""
    from native_sparse_attention_triton_b200 import ops

    pages, rows = 4 * 16 * 2 * 128, 3 * 2 * 128
    arena = torch.randn(2 * pages + 2 * rows, device="cuda").to(BF)
    kp, vp = (arena[i * pages:(i + 1) * pages].view(4, 16, 2, 128) for i in range(2))
    k, v = (arena[2 * pages + i * rows:2 * pages + (i + 1) * rows].view(3, 2, 128) for i in range(2))
    table, held = _ints([[0], [1], [2]]), _ints([0, 5, 15])
    k0, v0, rows_k, rows_v = kp.clone(), vp.clone(), k.clone(), v.clone()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    after = ops.paged_kv_append(kp, vp, table, held, k, v)
    assert torch.cuda.max_memory_allocated() - before <= 512  # the lengths
    for b, j in enumerate((0, 5, 15)):
        k0[b, j], v0[b, j] = rows_k[b], rows_v[b]
    assert after.tolist() == [1, 6, 16] and torch.equal(kp, k0) and torch.equal(vp, v0)
