"""cu_seqlens that do not fit the rows: nothing outside of the tensors is written, and the device status says so."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

N, HQ, HKV, GUARD = 300, 8, 2, 64
BIG = 2 ** 31 - 1
# and the lengths that the rows allow for, where there are such
CASES = [([0, 130, 330], [0, 130, 300]), ([0, N, 700], [0, N, N]), ([0, BIG], [0, N]), ([0, 100, 5000, 5100], [0, 100, N, N]), ([0, 130, -5], None),
         ([-7, N], None), ([-BIG, N], None), ([0, 250, 100, BIG], None), ([0, -100, 400], None), ([BIG, BIG], None), ([400, 500], None)]


class Guarded:
    """A tensor of `shape` between two stretches of a value that nothing else writes."""

    def __init__(self, shape, dtype):
        n, size = math.prod(shape), GUARD * 1024
        self.buf = torch.full((n + 2 * size,), 77, dtype=dtype, device="cuda")
        self.t, self.size = self.buf[size:size + n].view(shape), size

    def whole(self):
        return bool((self.buf[:self.size] == 77).all() and (self.buf[-self.size:] == 77).all())


@pytest.mark.parametrize("cu,fits", CASES)
@pytest.mark.parametrize("window,sinks,d", [(40, 3, 128), (0, 200, 64), (1000, 0, 128)])
def test_lengths_beyond_the_rows(cu, fits, window, sinks, d):
    from native_sparse_attention_triton_b200 import _lib, device_status

    lib, dtype = _lib.lib(), torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, do = [torch.randn(N, h, d, generator=g, device="cuda").to(dtype) for h in (HQ, HKV, HKV, HQ)]
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    strides = lambda *ts: _lib.strides_array(*[s for t in ts for s in t.stride()[:2]])

    def run(lengths):
        c = torch.tensor(lengths, dtype=torch.int32).cuda()
        o, rest, dq = [Guarded((N, HQ, d), dtype) for _ in range(3)]
        dk, dv = [Guarded((N, HKV, d), dtype) for _ in range(2)]
        lse = Guarded((N, HQ), torch.float32)
        size = lib.nsa_sink_window_attn_bwd_workspace(N, HQ, HKV, d)
        ws = Guarded((size,), torch.uint8)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.nsa_sink_window_attn_fwd(p(q), p(k), p(v), p(c), p(o.t), p(rest.t), p(lse.t), N, len(lengths) - 1, HQ, HKV, d, window, sinks,
                                            strides(q, k, v, o.t), d ** -0.5, 0, stream) == 0
        first = device_status()
        assert lib.nsa_sink_window_attn_bwd(p(q), p(k), p(v), p(o.t), p(rest.t), p(do), p(lse.t), p(c), p(dq.t), p(dk.t), p(dv.t), p(ws.t), size, N,
                                            len(lengths) - 1, HQ, HKV, d, window, sinks, strides(q, k, v, o.t, do, dq.t, dk.t, dv.t), d ** -0.5, 0,
                                            stream) == 0
        status = (first, device_status())
        assert all(x.whole() for x in (o, rest, dq, dk, dv, lse, ws))
        return status, [x.t for x in (o, dq, dk, dv)]

    status, got = run(cu)
    assert status == (2, 2)
    if fits:
        status, want = run(fits)
        assert status == (0, 0)
        for x, y in zip(got, want):
            # (dK and dV of some rows are sums whose order may differ)
            assert torch.allclose(x.float(), y.float(), rtol=2 ** -6, atol=1e-5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
