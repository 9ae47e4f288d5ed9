"""The paged cache's operators against their definitions in 64 bits."""
import pytest
import torch

from tests.sink_paged_refs import DECODE_SLACK, assert_within, evict_rows, paged_decode, rows_of

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Cache:
    """Random pages; a table of shuffled pages with -1 (or any number) where a sequence holds no row."""

    def __init__(self, lens, hkv, d, page, dtype, seed=0, spare=3, columns=None, heads_first=False, unused=-1, rows=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [(n + page - 1) // page for n in (rows or lens)]
        self.pages = sum(need) + spare
        shape = (self.pages, hkv, page, d) if heads_first else (self.pages, page, hkv, d)
        mk = lambda: torch.randn(*shape, generator=g, device="cuda").to(dtype)
        self.k, self.v = (mk().transpose(1, 2) if heads_first else mk() for _ in range(2))
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), columns or max(1, max(need))), unused, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.free, self.lens, self.seqlens, self.page, self.g = order[at:], list(lens), _ints(lens), page, g

    def queries(self, hq):
        return (torch.randn(len(self.lens), hq, self.k.shape[3], generator=self.g, device="cuda") * 2).to(self.k.dtype)


def _check_decode(c, hq, window=None, sinks=0, weights=False, scale=None):
    from native_sparse_attention_triton_b200 import device_status, ops

    q = c.queries(hq)
    cap = c.table.shape[1] * c.page
    w = torch.rand(len(c.lens), c.k.shape[2], cap + 5, device="cuda") if weights else None
    before = w.clone() if weights else None
    o = ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens, scale, window, sinks, w)
    value, bound, added = paged_decode(q, c.k, c.v, c.table, c.lens, window, sinks, scale)
    assert o.dtype == q.dtype
    assert_within(o, value, bound, "o")
    if weights:
        for b, (rows, p) in enumerate(added):
            want = before[b].double()
            want[:, rows] += p
            tol = torch.zeros_like(want)
            # the sum of at most 16 probabilities, and the rounding of the running sum
            tol[:, rows] = DECODE_SLACK * p + torch.finfo(torch.float32).eps * want[:, rows]
            assert ((w[b].double() - want).abs() <= tol).all(), b
    assert device_status() == 0


@pytest.mark.parametrize("d,dtype", [(128, BF), (128, FP), (64, BF), (64, FP)])
@pytest.mark.parametrize("page", [1, 7, 16, 64, 100, 256])
def test_pages(d, dtype, page):
    _check_decode(Cache([1, 31, 32, 33, 64, 65, 200, 0, 517], 2, d, page, dtype), 8)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (16, 1), (12, 4), (7, 7), (26, 2), (32, 8), (64, 4)])
@pytest.mark.parametrize("weights", [False, True])
def test_head_layouts(hq, hkv, weights):
    _check_decode(Cache([333, 5, 1200], hkv, 128, 16, BF), hq, weights=weights)


@pytest.mark.parametrize("lens", [[1], [2], [40000], [20000, 3, 9000], [0], [0, 0, 7], [100] * 600, [(i * 37) % 300 for i in range(333)]])
@pytest.mark.parametrize("d", [64, 128])
def test_lengths(lens, d):
    _check_decode(Cache(lens, 2, d, 32, BF), 4, weights=len(lens) < 10)


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 1), (0, 4), (1, 1), (31, 1), (32, 0), (99, 33), (99, 64), (700, 3), (10 ** 9, 4), (5, 10 ** 9)])
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
def test_window_and_sinks(window, sinks, d, dtype):
    _check_decode(Cache([0, 1, 2, 33, 100, 101, 164, 900, 5000], 2, d, 16, dtype), 8, window, sinks, weights=True)


def test_a_scale_of_its_own_and_a_wide_table():
    _check_decode(Cache([70, 500], 2, 128, 16, BF, columns=200), 8, scale=0.25)
    _check_decode(Cache([70, 500], 2, 128, 16, BF), 8, scale=-0.1)


@pytest.mark.parametrize("d", [64, 128])
def test_strides(d):
    """Pages with their heads outermost; K and V as halves of one tensor; a table and queries that are slices."""
    from native_sparse_attention_triton_b200 import ops

    c = Cache([300, 45, 61], 4, d, 32, BF, heads_first=True)
    _check_decode(c, 8, weights=True)
    both = torch.stack([c.k, c.v], 1).contiguous()
    wide = torch.full((3, 2 * c.table.shape[1]), -7, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    c.k, c.v, c.table = both[:, 0], both[:, 1], wide[:, :c.table.shape[1]]
    _check_decode(c, 8, 50, 3, weights=True)
    c.k = c.k[:, :, 1:2].expand(-1, -1, 4, -1)  # one head's keys for all heads
    _check_decode(c, 8, weights=True)
    q = torch.randn(3, 16, d, device="cuda").to(BF)[:, ::2]
    value, bound, _ = paged_decode(q, c.k, c.v, c.table, c.lens)
    assert_within(ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens), value, bound)


def test_a_long_cache_whose_offsets_pass_32_bits():
    """Rows at element offsets past 2^31, and page numbers up to 2^17, in a cache of 5 GB each."""
    from native_sparse_attention_triton_b200 import ops

    pages, page, hkv, d = 1 << 17, 16, 10, 128
    k, v = (torch.zeros(pages, page, hkv, d, dtype=BF, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    table = torch.tensor([[pages - 1, 5, pages - 2], [pages - 3, pages - 4, 0]], dtype=torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in table.flatten().tolist():
        k[t], v[t] = torch.randn(2, page, hkv, d, generator=g, device="cuda").to(BF)
    q = torch.randn(2, 20, d, generator=g, device="cuda").to(BF)
    value, bound, _ = paged_decode(q, k, v, table, [45, 30])
    assert_within(ops.paged_attention_decode(q, k, v, table, _ints([45, 30])), value, bound)
    rows = torch.randn(2, hkv, d, generator=g, device="cuda").to(BF)
    after = ops.paged_kv_append(k, v, table, _ints([45, 30]), rows, -rows)
    assert after.tolist() == [46, 31]
    assert torch.equal(k[pages - 2, 13], rows[0]) and torch.equal(v[pages - 4, 14], -rows[1])
    w = torch.rand(2, hkv, 48, generator=g, device="cuda")
    _, _, kept = ops.paged_kv_evict(k, v, table, _ints([45, 30]), w, _ints([[pages - 9], [3]]), 16, 1, 2)
    for b, page_to in enumerate((pages - 9, 3)):
        for h in range(hkv):
            assert torch.equal(k[page_to, :, h], rows_of(k, table[b], 45)[kept[b, h].long(), h])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_are_not_visible_may_be_anything(bad):
    """Slots behind a sequence's last row, pages of no sequence, rows between the sinks and the window."""
    c = Cache([70, 33, 5], 2, 128, 32, BF)
    for x in (c.k, c.v):
        x[c.free.long()] = bad
        for b, n in enumerate(c.lens):
            x[c.table[b, (n - 1) // 32].long(), (n - 1) % 32 + 1:] = bad
    _check_decode(c, 8, weights=True)
    for x in (c.k, c.v):
        x[c.table[0, 0].long(), 2:] = bad  # rows 2 .. 31 of the first sequence
    c.lens, c.seqlens, c.table = c.lens[:1], c.seqlens[:1], c.table[:1]
    _check_decode(c, 8, 30, 2, weights=True)


def test_page_numbers_outside_the_cache():
    """Rows on such pages count as not visible, and the device status says so."""
    from native_sparse_attention_triton_b200 import device_status, ops

    c = Cache([96, 40], 2, 128, 32, BF)
    q = c.queries(8)
    want, _, _ = paged_decode(q, c.k, c.v, c.table[:, ::2].contiguous(), [64, 0])
    table = c.table.clone()
    table[0, 1], table[1, 0], table[1, 1] = c.pages, -1, 2 ** 30
    o = ops.paged_attention_decode(q, c.k, c.v, table, c.seqlens)
    assert device_status() == 2
    assert (o.double() - want).abs().max() < 0.02 and (o[1] == 0).all()
    k0, v0 = c.k.clone(), c.v.clone()
    rows = torch.zeros(2, 2, 128, dtype=BF, device="cuda")
    ops.paged_kv_append(c.k, c.v, table, _ints([40, 0]), rows, rows)
    assert device_status() == 2 and torch.equal(c.k, k0) and torch.equal(c.v, v0)
    after = ops.paged_kv_append(c.k, c.v, c.table, _ints([96, -3]), rows, rows)  # no room left; a length below zero
    assert device_status() == 2 and torch.equal(c.k, k0) and after[0] == 96
    ops.paged_attention_decode(q, c.k, c.v, c.table, _ints([97, 1]))  # longer than its pages
    assert device_status() == 2
    ops.paged_kv_evict(c.k, c.v, table, c.seqlens, torch.rand(2, 2, 96, device="cuda"), _ints([[-5], [c.pages]]), 32, 0, 0)
    assert device_status() == 2 and torch.equal(c.k, k0) and torch.equal(c.v, v0)


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("held,new", [([0], [1]), ([5, 0, 31, 32, 63], [1] * 5), ([0, 3, 60, 9], [100, 0, 70, 1]), ([0] * 40, [(i * 5) % 9 for i in range(40)]),
                                      ([17], [2000])])
@pytest.mark.parametrize("page", [5, 32])
def test_append(d, dtype, held, new, page):
    from native_sparse_attention_triton_b200 import device_status, ops

    c = Cache(held, 3, d, page, dtype, rows=[a + b for a, b in zip(held, new)])
    n = sum(new)
    k, v = (torch.randn(n + 4, 3, d, generator=c.g, device="cuda").to(dtype) for _ in range(2))  # four rows behind the last sequence
    k0, v0 = c.k.clone(), c.v.clone()
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    after = ops.paged_kv_append(c.k, c.v, c.table, c.seqlens, k, v, _ints(cu))
    assert after.tolist() == [a + b for a, b in zip(held, new)] and c.seqlens.tolist() == held
    for b in range(len(held)):
        for j in range(new[b]):
            pos = held[b] + j
            at = (int(c.table[b, pos // page]), pos % page)
            k0[at], v0[at] = k[cu[b] + j], v[cu[b] + j]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
    if set(new) == {1}:  # the same without cu_seqlens
        c.k.zero_(), c.v.zero_()
        ops.paged_kv_append(c.k, c.v, c.table, c.seqlens, k[:n], v[:n])
        for b, pos in enumerate(held):
            at = (int(c.table[b, pos // page]), pos % page)
            assert torch.equal(c.k[at], k[b]) and torch.equal(c.v[at], v[b])
    assert device_status() == 0


def test_append_with_strides():
    from native_sparse_attention_triton_b200 import ops

    c = Cache([10, 3], 2, 128, 8, BF, heads_first=True, rows=[11, 4])
    kv = torch.randn(2, 4, 128, device="cuda").to(BF)
    k0, v0 = c.k.clone(), c.v.clone()
    odd = torch.randn(2 * 2 * 128 + 1, device="cuda").to(BF)[1:].view(2, 2, 128)  # an odd address: copied
    ops.paged_kv_append(c.k, c.v, c.table, c.seqlens, kv[:, :2], odd.clone())
    for b, pos in enumerate((10, 3)):
        at = (int(c.table[b, pos // 8]), pos % 8)
        k0[at], v0[at] = kv[b, :2], odd[b]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)


def _check_evict(lens, hkv, d, page, dtype, budget, sinks, recent, weights=None, extra=0, heads_first=False):
    from native_sparse_attention_triton_b200 import device_status, ops

    to = [(min(n, budget) + page - 1) // page for n in lens]
    c = Cache(lens, hkv, d, page, dtype, spare=sum(to) + 2, heads_first=heads_first)
    cap = c.table.shape[1] * page
    w = torch.rand(len(lens), hkv, cap + extra, generator=c.g, device="cuda") if weights is None else weights(len(lens), hkv, cap + extra)
    columns = -(-min(budget, cap) // page)
    target, at = torch.full((len(lens), columns), -1, dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(to):
        target[b, :n] = c.free[at:at + n]
        at += n
    k0, v0 = c.k.clone(), c.v.clone()
    after, sums, kept = ops.paged_kv_evict(c.k, c.v, c.table, c.seqlens, w, target, budget, sinks, recent)
    assert after.tolist() == [min(n, budget) for n in lens]
    assert sums.shape == w.shape and kept.shape == (len(lens), hkv, budget)
    for b, n in enumerate(lens):
        m = min(n, budget)
        for h in range(hkv):
            rows = evict_rows(w[b, h, :n].cpu(), n, budget, sinks, recent)
            assert kept[b, h].tolist() == rows + [-1] * (budget - m), (b, h)
            r = torch.tensor(rows, dtype=torch.long, device="cuda")
            assert torch.equal(sums[b, h, :m].view(torch.int32), w[b, h, r].view(torch.int32)) and (sums[b, h, m:] == 0).all()
            i = torch.arange(m, device="cuda")
            page_to = target[b].long()[i // page]
            k_old, v_old = rows_of(k0, c.table[b], n)[r, h], rows_of(v0, c.table[b], n)[r, h]
            k0[page_to, i % page, h], v0[page_to, i % page, h] = k_old, v_old
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)  # and nothing else was written
    assert device_status() == 0


@pytest.mark.parametrize("d,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("lens,page,budget,sinks,recent", [
    ([40], 16, 39, 0, 0), ([40], 16, 1, 0, 0), ([40], 16, 1, 1, 0), ([40], 16, 1, 0, 1), ([700, 3, 0, 512, 513], 16, 512, 4, 100),
    ([700, 30], 7, 300, 100, 200), ([5, 9], 8, 50, 1, 1), ([3000, 1600, 100], 64, 1024, 4, 0), ([1025], 32, 1024, 0, 1000)])
def test_evict(d, dtype, lens, page, budget, sinks, recent):
    _check_evict(lens, 3, d, page, dtype, budget, sinks, recent, extra=3)


def test_evict_a_long_sequence_and_strided_pages():
    _check_evict([30000], 1, 128, 64, BF, 5000, 4, 64)
    _check_evict([200, 90], 4, 64, 16, BF, 64, 2, 8, heads_first=True)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "negative", "nan", "inf", "tiny"])
def test_evict_weights_of_every_kind(kind):
    """Ties go to the lower row; both zeros are one; NaN counts as the smallest."""
    def make(*shape):
        g = torch.Generator(device="cuda").manual_seed(5)
        x = torch.rand(*shape, generator=g, device="cuda")
        if kind == "equal":
            return torch.full_like(x, 0.25)
        if kind == "few":
            return (x * 3).floor()
        if kind == "zeros":
            return torch.where(x < 0.5, 0.0, -0.0)
        if kind == "negative":
            return x - 0.5
        if kind == "nan":
            return torch.where(x < 0.7, float("nan"), x)
        if kind == "inf":
            return torch.where(x < 0.3, float("inf"), torch.where(x < 0.6, -float("inf"), x))
        return x * 1e-44

    _check_evict([1500, 700], 2, 64, 32, BF, 600, 3, 50, weights=make)


def test_shared_pages_and_a_repeated_sequence():
    """Two sequences with the same first pages, and the same sequence twice."""
    c = Cache([100, 100, 100], 2, 128, 16, BF)
    c.table[1, :4] = c.table[0, :4]
    c.table[2] = c.table[0]
    _check_decode(c, 8, weights=True)


def test_captured_calls_and_other_streams():
    """Two graphs captured one after the other and eager calls between their replays: each has a workspace of its own."""
    from native_sparse_attention_triton_b200 import device_status, ops

    a, b = Cache([5000, 100], 2, 128, 16, BF, seed=1, rows=[5001, 101]), Cache([900] * 40, 4, 64, 32, BF, seed=2)
    qa, qb = a.queries(8), b.queries(8)
    w = torch.zeros(40, 4, b.table.shape[1] * 32, device="cuda")
    new = torch.randn(2, 2, 128, device="cuda").to(BF)
    side = torch.cuda.Stream()

    def step_a():
        lens = ops.paged_kv_append(a.k, a.v, a.table, a.seqlens, new, new)
        return ops.paged_attention_decode(qa, a.k, a.v, a.table, lens)

    def step_b():
        return ops.paged_attention_decode(qb, b.k, b.v, b.table, b.seqlens, weights=w)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_a(), step_b()
    torch.cuda.current_stream().wait_stream(side)
    w.zero_()
    graphs, outs = [], []
    for step in (step_a, step_b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step())
        graphs.append(graph)
    want_b, bound_b, added = paged_decode(qb, b.k, b.v, b.table, b.lens)
    for turn in range(3):
        with torch.no_grad():
            new.normal_()
        want_a = None
        graphs[0].replay()
        eager = ops.paged_attention_decode(qb, b.k, b.v, b.table, b.seqlens)
        graphs[1].replay()
        want_a, bound_a, _ = paged_decode(qa, a.k, a.v, a.table, [5001, 101])
        assert_within(outs[0], want_a, bound_a)
        assert_within(outs[1], want_b, bound_b)
        assert_within(eager, want_b, bound_b)
    total = torch.stack([x for _, x in added]) * 3
    assert ((w[:, :, :900].double() - total).abs() <= DECODE_SLACK * total + 1e-6).all() and (w[:, :, 900:] == 0).all()
    assert device_status() == 0


def test_the_same_call_gives_the_same_bits():
    from native_sparse_attention_triton_b200 import ops

    c = Cache([30000, 17, 4000], 2, 128, 16, BF)
    q = c.queries(16)
    w = [torch.zeros(3, 2, c.table.shape[1] * 16, device="cuda") for _ in range(6)]
    first = ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens, weights=w[0])
    for x in w[1:]:
        assert torch.equal(ops.paged_attention_decode(q, c.k, c.v, c.table, c.seqlens, weights=x), first)
        assert torch.equal(x, w[0])


def test_versions_count_what_is_written():
    from native_sparse_attention_triton_b200 import ops

    c = Cache([20], 2, 64, 16, BF, rows=[21])
    w = torch.zeros(1, 2, 32, device="cuda")
    versions = [x._version for x in (c.k, c.v, w)]
    ops.paged_kv_append(c.k, c.v, c.table, c.seqlens, c.k[0, :1].clone(), c.v[0, :1].clone())
    ops.paged_attention_decode(c.queries(4), c.k, c.v, c.table, c.seqlens, weights=w)
    assert [x._version for x in (c.k, c.v, w)] == [v + 1 for v in versions]
    with torch.inference_mode():
        z = torch.zeros(1, 2, 32, device="cuda")
        ops.paged_attention_decode(c.queries(4), c.k, c.v, c.table, c.seqlens, weights=z)
        assert float(z.sum()) == pytest.approx(4, rel=1e-4)


def test_no_sequences():
    from native_sparse_attention_triton_b200 import ops

    c = Cache([5], 2, 64, 16, BF)
    table, lens = c.table[:0], c.seqlens[:0]
    rows = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    assert ops.paged_kv_append(c.k, c.v, table, lens, rows, rows).shape == (0,)
    assert ops.paged_attention_decode(torch.zeros(0, 4, 64, dtype=BF, device="cuda"), c.k, c.v, table, lens).shape == (0, 4, 64)
    w = torch.zeros(0, 2, 16, device="cuda")
    assert ops.paged_kv_evict(c.k, c.v, table, lens, w, table, 4, 0, 0)[2].shape == (0, 2, 4)
