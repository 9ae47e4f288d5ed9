"""What the rounding of the output took away, kept by the forward for the backward pass: gradients with it, within bounds that gradients without
it exceed.

dS = P (dO v - sum_d o dO) scale.  The output's gradient is chosen against the output's rounding: dO = sign(o - its 16-bit value), so that a sum
over the 16-bit o is off by sum_d |o - its 16-bit value|, about D h |o| / 3, all of one sign.  The forward's o with its rest is off by h * h of
the mass sum_j P |v| (two parts of each P, two of o) and by u = the least step of the type for each part, and by the 32-bit arithmetic.  No tile
of these cases is seen in full by all its rows (fewer than 64 keys), so that all exponentials come from the exponential unit: EXACT, 6e-5, is the
bound of the decode kernel's, 2^-22 of the unit and the fp32 sums of a logit."""
import ctypes
import math

import pytest
import torch

from tests.sink_paged_refs import assert_within, half_step, least_step, window_mask

pytestmark = pytest.mark.gpu

EXACT = 6e-5


def _strides(_lib, *tensors):
    return _lib.strides_array(*[s for t in tensors for s in t.stride()[:2]])


def _gradients(q, k, v, do, o, lse, rest, cu, window, sinks):
    from native_sparse_attention_triton_b200 import _lib

    lib, (n, hq, d), hkv = _lib.lib(), q.shape, k.shape[1]
    out = [torch.empty_like(x) for x in (q, k, v)]
    size = lib.nsa_sink_window_attn_bwd_workspace(n, hq, hkv, d)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
    code = 0 if q.dtype == torch.bfloat16 else 1
    rc = lib.nsa_sink_window_attn_bwd(p(q), p(k), p(v), p(o), p(rest), p(do), p(lse), p(cu), *map(p, out), p(ws), size, n, cu.numel() - 1, hq, hkv, d,
                                      window, sinks, _strides(_lib, q, k, v, o, do, *out), 1 / math.sqrt(d), code,
                                      ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 1, 128), (4, 4, 64), (6, 3, 64)])
@pytest.mark.parametrize("lens,window,sinks", [([60, 3, 33, 50], 0, 1), ([59, 60, 40], 3, 0), ([50] * 7, 2, 2)])
def test_gradients_with_and_without_it(dtype, hq, hkv, d, lens, window, sinks):
    from native_sparse_attention_triton_b200 import _lib, device_status

    n, g, scale = sum(lens), hq // hkv, 1 / math.sqrt(d)
    gen = torch.Generator(device="cuda").manual_seed(11)
    mk = lambda h, s=1.0: (torch.randn(n, h, d, generator=gen, device="cuda") * s).to(dtype)
    q, k, v = mk(hq, 2.0), mk(hkv), mk(hkv)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()
    o, rest, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(n, hq, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    rc = _lib.lib().nsa_sink_window_attn_fwd(p(q), p(k), p(v), p(cu), p(o), p(rest), p(lse), n, len(lens), hq, hkv, d, window, sinks,
                                             _strides(_lib, q, k, v, o), scale, 0 if dtype == torch.bfloat16 else 1,
                                             ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    h, u = half_step(dtype), least_step(dtype)
    exact, parts = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda"), []
    start = 0
    for m in lens:
        see = window_mask(m, window, sinks, "cuda")
        for head in range(hq):
            part = slice(start, start + m)
            prob = torch.softmax((q[part, head].double() @ k[part, head // g].double().T * scale).masked_fill(~see, -math.inf), 1)
            exact[part, head] = prob @ v[part, head // g].double()
            parts.append((part, head, see, prob))
        start += m
    do = torch.where(exact >= o.double(), 1.0, -1.0).to(dtype)
    value = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k)]
    bound = [torch.zeros_like(x) for x in value]
    for part, head, see, prob in parts:
        qh, kh, vh, gh = q[part, head].double(), k[part, head // g].double(), v[part, head // g].double(), do[part, head].double()
        dp, delta = gh @ vh.T, (exact[part, head] * gh).sum(1, keepdim=True)
        ds = prob * (dp - delta) * scale
        o_kept = (2 * h * h + EXACT) * (prob @ vh.abs()) + u * (2 + see.double() @ vh.abs())
        err = h * ds.abs() + u * see + prob * scale * ((o_kept * gh.abs()).sum(1, keepdim=True) + EXACT * (gh.abs() @ vh.abs().T + delta.abs()))
        value[0][part, head] = ds @ kh
        bound[0][part, head] = err @ kh.abs()
        value[1][part, head // g] += ds.T @ qh
        bound[1][part, head // g] += err.T @ qh.abs()
    for x, t in zip(value, bound):
        t += h * x.abs() * (1 + h) + u
    dq, dk, _ = _gradients(q, k, v, do, o, lse, rest, cu, window, sinks)
    assert_within(dq, value[0], bound[0], "dq")
    assert_within(dk, value[1], bound[1], "dk")
    if dtype == torch.bfloat16:  # (fp16: h is no more than 8 times EXACT)
        dq, dk, _ = _gradients(q, k, v, do, o, lse, None, cu, window, sinks)
        for got, x, t in zip((dq, dk), value, bound):
            assert ((got.double() - x).abs() > t).double().mean() > 0.01
    assert device_status() == 0
