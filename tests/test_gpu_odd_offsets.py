"""Inputs that are contiguous as torch sees it but not laid out as the kernels read rows: views at an odd offset, and one row with an odd stride.
They are copied, and the results are those of aligned tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _odd(t):
    """The same values at an address that is no multiple of 16 bytes."""
    flat = torch.empty(t.numel() + 3, dtype=t.dtype, device=t.device)[3:]
    flat.copy_(t.flatten())
    x = flat.view(t.shape)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


def _odd_stride(t):
    """One row whose stride to a next one is odd."""
    assert t.shape[0] == 1
    x = t.as_strided(t.shape, (t.numel() + 3, *t.stride()[1:]))
    assert x.is_contiguous()
    return x


def _calls(rows):
    from native_sparse_attention_triton_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(rows)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    q, k, v = mk(rows, 8, 128), mk(rows, 2, 128), mk(rows, 2, 128)
    cu = torch.tensor([0, rows], dtype=torch.int32).cuda()
    kp, vp = mk(4, 16, 2, 128), mk(4, 16, 2, 128)
    table = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None].contiguous()
    held = torch.full((rows,), 7, dtype=torch.int32, device="cuda")
    kc, vc = mk(rows, 50, 2, 128), mk(rows, 50, 2, 128)
    lens = torch.full((rows,), 33, dtype=torch.int32, device="cuda")

    def append(a, b):
        x, y = kp.clone(), vp.clone()
        ops.paged_kv_append(x, y, table, held, a, b)
        return torch.stack([x, y])

    return {
        "sink_window_attention": ([q, k, v], lambda a, b, c: ops.sink_window_attention(a, b, c, cu, 20, 2)),
        "sliding_window_attention": ([q, k, v], lambda a, b, c: ops.sliding_window_attention(a, b, c, cu, rows, 20)),
        "flash_attention_varlen": ([q, k, v], lambda a, b, c: ops.flash_attention_varlen(a, b, c, cu, cu, rows, rows, True)),
        "flash_attention_decode": ([q], lambda a: ops.flash_attention_decode(a, kc, vc, lens)),
        "paged_attention_decode": ([q], lambda a: ops.paged_attention_decode(a, kp, vp, table, held)),
        "paged_kv_append": ([k, v], append),
    }


NAMES = ["sink_window_attention", "sliding_window_attention", "flash_attention_varlen", "flash_attention_decode", "paged_attention_decode", "paged_kv_append"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("rows,change", [(1, _odd), (3, _odd), (1, _odd_stride)])
def test_they_are_copied(name, rows, change):
    args, call = _calls(rows)[name]
    want = call(*args)
    for i in range(len(args)):
        assert torch.equal(call(*[change(x) if i == j else x for j, x in enumerate(args)]), want)


def test_gradients_of_leaves_at_odd_offsets():
    from native_sparse_attention_triton_b200 import ops

    args, call = _calls(3)["sink_window_attention"]
    do = torch.ones_like(args[0])
    grads = []
    for change in (lambda x: x.clone(), _odd):
        leaves = [change(x).requires_grad_(True) for x in args]
        grads.append(torch.autograd.grad([call(*leaves)], leaves, [change(do)]))
    for a, b in zip(*grads):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=1e-5)


def test_a_cache_is_filled_from_rows_at_odd_offsets():
    from native_sparse_attention_triton_b200.kv_cache import inner_contiguous

    x = torch.randn(2, 2, 128, device="cuda").to(BF)
    y = inner_contiguous(_odd(x))
    assert y.data_ptr() % 16 == 0 and torch.equal(x, y)
    assert inner_contiguous(x) is x
