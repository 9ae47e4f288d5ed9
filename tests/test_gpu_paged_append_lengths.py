"""paged_kv_append behind lengths that no table has room for."""
import pytest
import torch

from tests.test_gpu_paged import BF, Cache, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, 64])
def test_lengths_up_to_the_type_s_largest(held):
    """Their rows are dropped, the lengths after that are the capacity, and the status says so."""
    from native_sparse_attention_triton_b200 import device_status, ops

    c = Cache([64, 3], 2, 128, 32, BF, rows=[64, 40])
    k0, v0 = c.k.clone(), c.v.clone()
    rows = torch.randn(2, 2, 128, device="cuda").to(BF)
    after = ops.paged_kv_append(c.k, c.v, c.table, _ints([held, 3]), rows, rows)
    assert after.tolist() == [64, 4] and device_status() == 2
    at = (int(c.table[1, 0]), 3)
    k0[at], v0[at] = rows[1], rows[1]
    many = torch.randn(12, 2, 128, device="cuda").to(BF)
    after = ops.paged_kv_append(c.k, c.v, c.table, _ints([held, 4]), many, many, _ints([0, 10, 12]))
    assert after.tolist() == [64, 6] and device_status() == 2
    for j in range(2):
        at = (int(c.table[1, 0]), 4 + j)
        k0[at], v0[at] = many[10 + j], many[10 + j]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
