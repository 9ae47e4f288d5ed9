"""The operators together, as a server with a window, sinks and a bounded cache runs them: a prompt's attention and its rows into the cache,
tokens one at a time with account of their weights, an eviction, more tokens."""
import pytest
import torch

from tests.sink_paged_refs import assert_within, evict_rows, paged_decode, rows_of, sink_window

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_prompt_steps_eviction_steps(d, dtype):
    from native_sparse_attention_triton_b200 import device_status, ops

    lens, steps, hq, hkv, page, window, sinks = [150, 37, 260], 6, 8, 2, 16, 90, 4
    g = torch.Generator(device="cuda").manual_seed(0)
    total = [n + steps for n in lens]
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    q, k, v = [[mk(n, h, d) for n in total] for h in (hq, hkv, hkv)]  # whole sequences, prompt and tokens to come
    cu = torch.tensor([0, 150, 187, 447], dtype=torch.int32).cuda()
    prompt = lambda x: torch.cat([t[:n] for t, n in zip(x, lens)])

    columns = (max(total) + steps + page - 1) // page
    pool = torch.randperm(6 * columns, generator=g, device="cuda").to(torch.int32)
    kp, vp = mk(6 * columns, page, hkv, d), mk(6 * columns, page, hkv, d)
    table, fresh = pool[:3 * columns].view(3, columns), pool[3 * columns:].view(3, columns)

    # what every position of the whole sequences sees, in one call
    whole = ops.sink_window_attention(torch.cat(q), torch.cat(k), torch.cat(v), torch.tensor([0] + total, dtype=torch.int32).cumsum(0).int().cuda(),
                                      window, sinks)
    value, bound = sink_window(torch.cat(q), torch.cat(k), torch.cat(v), total, window, sinks)
    assert_within(whole, value[0], bound[0])

    o = ops.sink_window_attention(prompt(q), prompt(k), prompt(v), cu, window, sinks)
    seqlens = ops.paged_kv_append(kp, vp, table, torch.zeros(3, dtype=torch.int32, device="cuda"), prompt(k), prompt(v), cu)
    at, first = 0, 0
    for n, t in zip(lens, total):
        assert_within(o[at:at + n], value[0][first:first + n], bound[0][first:first + n])
        at, first = at + n, first + t
    weights = torch.zeros(3, hkv, columns * page, device="cuda")
    for i in range(steps):
        row = lambda x: torch.stack([t[n + i] for t, n in zip(x, lens)])
        seqlens = ops.paged_kv_append(kp, vp, table, seqlens, row(k), row(v))
        o = ops.paged_attention_decode(row(q), kp, vp, table, seqlens, window_size=window, num_sinks=sinks, weights=weights)
        first = 0
        for b, (n, t) in enumerate(zip(lens, total)):
            assert_within(o[b], value[0][first + n + i], bound[0][first + n + i])
            first += t
    assert seqlens.tolist() == total
    # every step hands out one unit for each query head
    assert torch.allclose(weights.sum((1, 2)), torch.full((3,), float(steps * hq), device="cuda"), rtol=1e-4)

    budget, recent = 64, 20
    kept_rows = [[evict_rows(weights[b, h, :n].cpu(), n, budget, sinks, recent) for h in range(hkv)] for b, n in enumerate(total)]
    seqlens, weights, kept = ops.paged_kv_evict(kp, vp, table, seqlens, weights, fresh, budget, sinks, recent)
    assert seqlens.tolist() == [min(n, budget) for n in total]
    for b, n in enumerate(total):
        for h in range(hkv):
            m = min(n, budget)
            assert kept[b, h, :m].tolist() == kept_rows[b][h]
            assert torch.equal(rows_of(kp, fresh[b], m)[:, h], k[b][kept_rows[b][h], h])
    new = [mk(3, hq, d), mk(3, hkv, d), mk(3, hkv, d)]
    seqlens = ops.paged_kv_append(kp, vp, fresh, seqlens, new[1], new[2])
    o = ops.paged_attention_decode(new[0], kp, vp, fresh, seqlens, weights=weights)
    want, tol, _ = paged_decode(new[0], kp, vp, fresh, [min(n, budget) + 1 for n in total])
    assert_within(o, want, tol)
    assert device_status() == 0
