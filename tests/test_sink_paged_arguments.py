"""Refusals of sink_window_attention and the paged operators, and the references they are tested against; no GPU."""
import pytest
import torch

from native_sparse_attention_triton_b200 import _lib, ops
from tests.sink_paged_refs import evict_rows, sink_window, window_mask

I = torch.int32


def _window(**change):
    a = dict(q=torch.zeros(10, 4, 128).bfloat16(), k=torch.zeros(10, 2, 128).bfloat16(), v=torch.zeros(10, 2, 128).bfloat16(),
             cu=torch.tensor([0, 10], dtype=I), window=4, sinks=1, scale=None)
    a.update(change)
    return ops.sink_window_attention(a["q"], a["k"], a["v"], a["cu"], a["window"], a["sinks"], a["scale"])


def test_sink_window_gets_as_far_as_the_device():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _window()


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(10, 4, 128)), dict(k=torch.zeros(10, 2, 128).half()), dict(q=torch.zeros(10, 4 * 128).bfloat16()),
    dict(q=torch.zeros(9, 4, 128).bfloat16()), dict(v=torch.zeros(10, 1, 128).bfloat16()), dict(q=torch.zeros(10, 3, 128).bfloat16()),
    dict(q=torch.zeros(10, 4, 64).bfloat16()), dict(cu=torch.tensor([0, 10])), dict(cu=torch.tensor([0], dtype=I)), dict(window=-1), dict(sinks=-1),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=1e-60), dict(scale=1e60), dict(cu=torch.tensor([[0, 10]], dtype=I)),
    {x: torch.zeros(10, 2, 96).bfloat16() for x in "qkv"}, dict(k=torch.zeros(10, 0, 128).bfloat16(), v=torch.zeros(10, 0, 128).bfloat16())])
def test_sink_window_refuses(change):
    with pytest.raises(AssertionError):
        _window(**change)


@pytest.mark.parametrize("heads", [6, 32 * 2])
def test_sink_window_groups_that_are_not_built(heads):
    with pytest.raises(NotImplementedError):
        _window(q=torch.zeros(10, heads, 128).bfloat16())


def _cache(**change):
    a = dict(kp=torch.zeros(6, 16, 2, 128).bfloat16(), vp=torch.zeros(6, 16, 2, 128).bfloat16(), table=torch.zeros(3, 2, dtype=I),
             seqlens=torch.tensor([5, 0, 20], dtype=I), k=torch.zeros(3, 2, 128).bfloat16(), v=torch.zeros(3, 2, 128).bfloat16(), cu=None,
             q=torch.zeros(3, 8, 128).bfloat16(), scale=None, window=None, sinks=0, weights=torch.zeros(3, 2, 32),
             target=torch.zeros(3, 1, dtype=I), budget=16, keep=1, recent=4)
    a.update(change)
    return a


CALLS = {
    "append": lambda a: ops.paged_kv_append(a["kp"], a["vp"], a["table"], a["seqlens"], a["k"], a["v"], a["cu"]),
    "decode": lambda a: ops.paged_attention_decode(a["q"], a["kp"], a["vp"], a["table"], a["seqlens"], a["scale"], a["window"], a["sinks"], a["weights"]),
    "evict": lambda a: ops.paged_kv_evict(a["kp"], a["vp"], a["table"], a["seqlens"], a["weights"], a["target"], a["budget"], a["keep"], a["recent"]),
}


@pytest.mark.parametrize("call", CALLS)
def test_paged_operators_get_as_far_as_the_device(call):
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        CALLS[call](_cache())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        CALLS[call](_cache(k=torch.zeros(7, 2, 128).bfloat16(), v=torch.zeros(7, 2, 128).bfloat16(), cu=torch.tensor([0, 1, 1, 7], dtype=I), window=3))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change", [
    dict(kp=torch.zeros(6, 16, 2, 128)), dict(vp=torch.zeros(6, 16, 2, 128).half()), dict(kp=torch.zeros(6, 32, 2, 128).bfloat16()),
    dict(kp=torch.zeros(6, 16, 2, 96).bfloat16(), vp=torch.zeros(6, 16, 2, 96).bfloat16()),
    dict(kp=torch.zeros(0, 16, 2, 128).bfloat16(), vp=torch.zeros(0, 16, 2, 128).bfloat16()), dict(table=torch.zeros(3, 2, dtype=torch.int64)),
    dict(table=torch.zeros(6, dtype=I)), dict(table=torch.zeros(2, 3, dtype=I).T), dict(table=torch.zeros(3, 0, dtype=I)),
    dict(seqlens=torch.zeros(3)), dict(seqlens=torch.zeros(2, dtype=I)), dict(kp=torch.zeros(6, 16, 128, 2).bfloat16().transpose(2, 3)),
    dict(kp=torch.zeros(6 * 16 * 2 * 128 + 1).bfloat16()[1:].view(6, 16, 2, 128)), dict(kp=torch.zeros(6, 16, 2, 132).bfloat16()[..., :128])])
def test_caches_that_are_refused(call, change):
    with pytest.raises(AssertionError):
        CALLS[call](_cache(**change))


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(3, 4, 128).bfloat16()), dict(k=torch.zeros(3, 2, 128).half(), v=torch.zeros(3, 2, 128).half()),
    dict(k=torch.zeros(4, 2, 128).bfloat16(), v=torch.zeros(4, 2, 128).bfloat16()), dict(cu=torch.tensor([0, 3], dtype=I)),
    dict(cu=torch.tensor([0, 1, 2, 3]))])
def test_rows_that_append_refuses(change):
    with pytest.raises(AssertionError):
        CALLS["append"](_cache(**change))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 8, 128).bfloat16()), dict(q=torch.zeros(3, 7, 128).bfloat16()), dict(q=torch.zeros(3, 8, 128).half()),
    dict(q=torch.zeros(3, 8, 64).bfloat16()), dict(window=-1), dict(sinks=-1), dict(scale=float("inf")), dict(scale=1e60),
    dict(weights=torch.zeros(3, 2, 31)), dict(weights=torch.zeros(3, 4, 32)), dict(weights=torch.zeros(3, 2, 32).half())])
def test_queries_that_decode_refuses(change):
    with pytest.raises(AssertionError):
        CALLS["decode"](_cache(**change))


def test_groups_that_decode_does_not_have():
    with pytest.raises(NotImplementedError):
        CALLS["decode"](_cache(q=torch.zeros(3, 34, 128).bfloat16()))


@pytest.mark.parametrize("change", [
    dict(weights=torch.zeros(3, 2, 31)), dict(weights=torch.zeros(3, 1, 32)), dict(weights=torch.zeros(3, 2, 32).double()),
    dict(weights=torch.zeros(3, 32, 2).transpose(1, 2)), dict(target=torch.zeros(3, 2)), dict(target=torch.zeros(2, 1, dtype=I)), dict(budget=0),
    dict(budget=17), dict(keep=-1), dict(recent=-1), dict(keep=10, recent=7), dict(keep=17)])
def test_evictions_that_are_refused(change):
    with pytest.raises(AssertionError):
        CALLS["evict"](_cache(**change))


@pytest.mark.parametrize("call", ["append", "evict"])
def test_caches_that_cannot_be_written(call):
    pages = torch.zeros(6, 16, 2, 128).bfloat16()
    for kp, vp in ((pages, pages), (pages.narrow(0, 0, 1).expand(6, 16, 2, 128), pages), (pages[:, :, :1].expand(6, 16, 2, 128), pages)):
        with pytest.raises(RuntimeError, match="unsupported operation"):
            CALLS[call](_cache(kp=kp, vp=vp))
    with pytest.raises(AssertionError):
        CALLS[call](_cache(kp=pages.clone().requires_grad_(True)))


def test_weights_that_cannot_be_added_to():
    with pytest.raises(RuntimeError, match="unsupported operation"):
        CALLS["decode"](_cache(weights=torch.zeros(3, 1, 32).expand(3, 2, 32)))
    with pytest.raises(AssertionError):
        CALLS["decode"](_cache(weights=torch.zeros(3, 2, 32, requires_grad=True)))


def test_c_interface_refuses_before_it_touches_a_device():
    lib = _lib.lib()
    z = _lib.strides_array(*[8] * 16)
    assert lib.nsa_sink_window_attn_fwd(*[None] * 7, 1, 1, 1, 1, 128, 1, 1, z, 1.0, 0, None) == -1
    assert lib.nsa_sink_window_attn_bwd(*[None] * 12, 0, 1, 1, 1, 1, 128, 1, 1, z, 1.0, 0, None) == -1
    assert lib.nsa_paged_kv_append(*[None] * 8, 1, 1, 1, 128, 1, 1, 1, z, None) == -1
    assert lib.nsa_paged_attn_decode(*[None] * 8, 0, 1, 1, 1, 128, 1, 1, 1, 0, 0, z, 1.0, 0, None) == -1
    assert lib.nsa_paged_kv_evict(*[None] * 9, 1, 1, 128, 1, 1, 1, 1, 1, 1, 0, 0, z, None) == -1
    p = 4096  # an address that is never followed: the sizes are refused first
    assert lib.nsa_paged_attn_decode(*[p] * 6, None, p, 0, 1, 1, 1, 128, 1, 1, 1, 0, 0, z, 1.0, 0, None) == -3      # scratch
    assert lib.nsa_paged_attn_decode(*[p] * 6, None, p, 1 << 40, 1, 17, 1, 128, 1, 1, 1, 0, 0, z, 1.0, 0, None) == -2
    assert lib.nsa_paged_kv_append(*[p] * 8, 1, 1, 1, 96, 1, 1, 1, z, None) == -2
    assert lib.nsa_paged_kv_evict(*[p] * 9, 1, 1, 128, 1, 1, 1, 1, 1, 4, 5, 0, z, None) == -1                       # sinks beyond the budget
    assert lib.nsa_sink_window_attn_fwd(*[p] * 7, 1, 1, 65536, 65536, 128, 1, 1, z, 1.0, 0, None) == -2                 # the grid's second dimension
    odd = _lib.strides_array(*[4] * 16)
    assert lib.nsa_sink_window_attn_fwd(*[p] * 7, 1, 1, 1, 1, 128, 1, 1, odd, 1.0, 0, None) == -1
    assert lib.nsa_sink_window_attn_bwd(*[p] * 12, 0, 1, 1, 1, 1, 128, 1, 1, z, 1.0, 0, None) == -3


def test_reference_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    lens, window, sinks = [7, 3], 2, 1
    x = [torch.randn(10, h, 4, generator=g).double() for h in (4, 2, 2, 4)]

    def loss(q, k, v):
        return (sink_window(q, k, v, lens, window, sinks)[0][0] * x[3]).sum()

    value, _ = sink_window(*x[:3], lens, window, sinks, x[3])
    for which in range(3):
        for at in [(0, 0, 0), (5, 1, 2), (9, 0, 3), (6, 1, 1)]:
            step = 1e-6
            up, down = [t.clone() for t in x[:3]], [t.clone() for t in x[:3]]
            up[which][at] += step
            down[which][at] -= step
            assert float((loss(*up) - loss(*down)) / (2 * step)) == pytest.approx(float(value[1 + which][at]), rel=1e-6, abs=1e-8)


def test_reference_mask_and_eviction():
    see = window_mask(6, 2, 1, "cpu")
    assert see.int().tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 0, 0], [1, 0, 1, 1, 1, 0], [1, 0, 0, 1, 1, 1]]
    w = torch.tensor([0.0, 5.0, 1.0, 5.0, float("nan"), 2.0, 0.0])
    assert evict_rows(w, 7, 4, 1, 1) == [0, 1, 3, 6]
    assert evict_rows(w, 7, 3, 1, 1) == [0, 1, 6]
    assert evict_rows(w, 3, 4, 1, 1) == [0, 1, 2]
