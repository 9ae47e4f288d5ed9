"""Attention with a sliding window and sinks, and a paged key-value cache with the operators that fill, read and shrink it.

Four operators, each computed two ways by ``run``: in a plain form of elementary torch operations in 32 bits (``own`` false), and through
the framework's entry points (``own`` true).

* ``window`` -- causal varlen attention where a query sees the last ``window`` keys, itself, and the first ``sinks`` keys of its
                sequence; forward alone (a prompt) or with its gradients (training);
* ``append`` -- rows of keys and values written behind the rows that a paged cache holds: one a sequence (decoding) or many (a prompt);
* ``decode`` -- one query token per sequence over the paged cache, all of it or a window and sinks; with ``weights`` the probabilities
                that each row received, summed over the heads of its group, are added to a running sum;
* ``evict``  -- of each sequence the first rows, the last ones and those with the largest running sums are kept, up to a budget, and
                written to other pages.

``draw()`` gives cases of the ranges that the listed ones stand for: 1 to 32 768 tokens, 1 to 256 sequences, pages of 8 to 256 rows, the head
layouts 64/4, 32/2, 32/4, 32/8, 16/2, 16/1 and 8/8, head_dim 64 and 128, bf16 and fp16.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------------ cases
def _text(lens):
    return ",".join(str(n) for n in lens)


def _window(lens, hq, hkv, window, sinks, train, d=128, dtype="bf16"):
    return dict(kind="window", lens=_text(lens), hq=hq, hkv=hkv, d=d, dtype=dtype, window=window, sinks=sinks, train=train)


def _append(held, new, hkv, page, d=128, dtype="bf16"):
    return dict(kind="append", lens=_text(held), new=_text(new), hkv=hkv, d=d, dtype=dtype, page=page)


def _decode(lens, hq, hkv, page, d=128, dtype="bf16", window=-1, sinks=0, weights=False):
    return dict(kind="decode", lens=_text(lens), hq=hq, hkv=hkv, d=d, dtype=dtype, page=page, window=window, sinks=sinks, weights=weights)


def _evict(lens, hkv, page, budget, sinks, recent, d=128, dtype="bf16"):
    return dict(kind="evict", lens=_text(lens), hkv=hkv, d=d, dtype=dtype, page=page, budget=budget, sinks=sinks, recent=recent)


def listed():
    named = [
        # fine-tuning on short samples: small kernels, launches and host time count
        ("window_short_samples", _window([200, 777], 32, 2, 128, 4, True)),
        # a packed training batch of ragged documents, the headline benchmark's heads and the layer's window
        ("window_packed_32k", _window([1024, 11743, 20001], 64, 4, 512, 4, True)),
        # prompts of a model with head_dim 64 and groups of four, fp16, read once with a wide window and many sinks
        ("window_prompts_head_dim_64", _window([333, 2500, 5000], 32, 8, 2048, 64, False, d=64, dtype="fp16")),
        # the new token's rows of a serving batch, one a sequence
        ("append_batch_76", _append([i * 37 % 76 * 13 + 1 for i in range(76)], [1] * 76, 4, 64)),
        # ragged prompts that go into the cache in one call, behind what a sequence holds already
        ("append_prompts_16k", _append([0, 300, 0, 77], [8192, 4000, 1, 4191], 8, 16)),
        # one short conversation: latency alone
        ("decode_one_short", _decode([517], 32, 2, 64)),
        # a serving batch of 1 to 8192 tokens, the lengths of the dense decode operators' self-test
        ("decode_batch_76", _decode([min(8192, i * 37 % 76 * 128 + 1) for i in range(76)], 32, 4, 64)),
        # a few long contexts, small pages
        ("decode_long_contexts", _decode([65536, 40001, 7, 98304], 64, 4, 16)),
        # many streams that see a window and sinks only
        ("decode_window_sinks", _decode([1 + i * 67 % 128 * 61 for i in range(128)], 32, 8, 32, d=64, dtype="fp16", window=1023, sinks=4)),
        # decoding that keeps account of what each row receives, for the eviction below
        ("decode_weights", _decode([1100 + i * 29 % 32 * 97 for i in range(32)], 32, 8, 64, weights=True)),
        # one conversation whose cache has grown a page past its budget
        ("evict_one_page", _evict([4160], 8, 64, 4096, 4, 512)),
        # that eviction of a batch: caches of 1100 to 4107 rows cut to 1024
        ("evict_batch_32", _evict([1100 + i * 29 % 32 * 97 for i in range(32)], 8, 64, 1024, 4, 256)),
    ]
    return [dict(name=n, **c) for n, c in named]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _split(rng, total, seqs):
    weights = [1.0] * seqs if rng.random() < 0.3 else [rng.uniform(0.02, 1.0) for _ in range(seqs)]
    return [max(1, int(total * w / sum(weights))) for w in weights]


def draw(rng):
    kind = rng.choice(["window", "window", "append", "decode", "decode", "evict"])
    hq, hkv = rng.choice([(64, 4), (32, 2), (32, 4), (32, 8), (16, 2), (16, 1), (8, 8)])
    d, dtype, page = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "fp16"]), rng.choice([8, 16, 16, 32, 48, 64, 64, 128, 256])
    if kind == "window":
        total = _log_uniform(rng, 1, 32768)
        lens = _split(rng, total, rng.choice([1, 1, 2, 3, 8]))
        window = rng.choice([0, _log_uniform(rng, 1, 64), _log_uniform(rng, 64, 512), 128, 512, _log_uniform(rng, 512, 4096)])
        train = rng.random() < 0.6
        while total * hq * window > 2 ** 30:
            window //= 2
        return _window(lens, hq, hkv, window, rng.choice([0, 1, 4, 4, 16, 64, rng.randint(1, 130)]), train, d, dtype)
    batch = _log_uniform(rng, 1, 256)
    if kind == "append":
        held = [rng.randint(0, 1024) for _ in range(batch)]
        new = [1] * batch if rng.random() < 0.5 else _split(rng, _log_uniform(rng, batch, 16384), batch)
        return _append(held, new, hkv, page, d, dtype)
    if kind == "decode":
        longest = _log_uniform(rng, 1, max(64, min(98304, 524288 // batch)))
        lens = [longest if rng.random() < 0.2 else rng.randint(1, longest) for _ in range(batch)]
        window = rng.choice([-1, -1, -1, 0, _log_uniform(rng, 1, 4096)])
        return _decode(lens, hq, hkv, page, d, dtype, window, rng.choice([0, 1, 4, 16]) if window >= 0 else 0, rng.random() < 0.3)
    longest = _log_uniform(rng, 32, max(64, min(16384, 131072 // batch)))
    lens = [longest if rng.random() < 0.3 else rng.randint(1, longest) for _ in range(batch)]
    budget = rng.randint(8, longest)
    sinks = rng.choice([0, 1, 4])
    return _evict(lens, hkv, page, budget, sinks, rng.randint(0, budget - sinks), d, dtype)


# ----------------------------------------------------------------------------------------------------------------- inputs
def _ints(text):
    return [int(n) for n in text.split(",")]


def _device(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _device(cu)


class _Maker:
    """Seeded tensors on the GPU."""

    def __init__(self, seed, dtype):
        self.g = torch.Generator(device=DEVICE).manual_seed(seed)
        self.dtype = dtype

    def normal(self, *shape, scale=1.0):
        if scale == 1.0:
            return torch.randn(*shape, generator=self.g, device=DEVICE, dtype=self.dtype)
        return (torch.randn(*shape, generator=self.g, device=DEVICE) * scale).to(self.dtype)

    def weights(self, *shape):
        """Running sums of probabilities: a few rows hold most of them, some have received nothing."""
        w = torch.rand(*shape, generator=self.g, device=DEVICE)
        return torch.where(w < 0.05, 0.0, w.square().square() * 8)

    def table(self, rows, page, spare=0):
        """Pages for `rows[b]` rows of each sequence out of a shuffled pool: (int32 table, pages in the pool)."""
        need = [(n + page - 1) // page for n in rows]
        total = sum(need) + spare
        pool = torch.randperm(total, generator=self.g, device=DEVICE).to(torch.int32)
        table = torch.zeros(len(rows), max(1, max(need)), dtype=torch.int32, device=DEVICE)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = pool[at:at + n]
            at += n
        return table, total, pool[at:]


def prepare(case, seed):
    c, m = case, _Maker(seed, DTYPES[case["dtype"]])
    lens = _ints(c["lens"])
    hkv, d = c["hkv"], c["d"]
    s = dict(c=c)
    if c["kind"] == "window":
        n = sum(lens)
        # queries of twice the usual size: rows that look at few keys, as trained models have them
        s.update(cu=_cu(lens), q=m.normal(n, c["hq"], d, scale=2.0), k=m.normal(n, hkv, d), v=m.normal(n, hkv, d))
        s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), torch.tensor(lens, device=DEVICE))
        if c["train"]:
            s["do"] = m.normal(n, c["hq"], d)
            s["leaves"] = [s[x].requires_grad_(True) for x in "qkv"]
        return s
    if c["kind"] == "append":
        new = _ints(c["new"])
        s["table"], pages, _ = m.table([a + b for a, b in zip(lens, new)], c["page"])
        s.update(held=_device(lens), cu=None if max(new) == min(new) == 1 else _cu(new), k=m.normal(sum(new), hkv, d), v=m.normal(sum(new), hkv, d))
        s["seq"] = torch.repeat_interleave(torch.arange(len(new), device=DEVICE), torch.tensor(new, device=DEVICE))
    elif c["kind"] == "decode":
        s["table"], pages, _ = m.table(lens, c["page"])
        s.update(lens=_device(lens), q=m.normal(len(lens), c["hq"], d, scale=2.0), weights=None)
        if c["weights"]:
            s["weights"] = m.weights(len(lens), hkv, s["table"].shape[1] * c["page"])
    else:
        kept = [min(n, c["budget"]) for n in lens]
        need = [(n + c["page"] - 1) // c["page"] for n in kept]
        s["table"], pages, free = m.table(lens, c["page"], sum(need))
        s["target"] = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEVICE)
        at = 0
        for b, n in enumerate(need):
            s["target"][b, :n] = free[at:at + n]
            at += n
        s.update(lens=_device(lens), weights=m.weights(len(lens), hkv, s["table"].shape[1] * c["page"]))
    s["kp"], s["vp"] = m.normal(pages, c["page"], hkv, d), m.normal(pages, c["page"], hkv, d)
    return s


# ------------------------------------------------------------------------------------------------------------------- runs
def run(state):
    c = state["c"]
    if own:
        return _own(c["kind"], c, state)
    return {"window": _plain_window, "append": _plain_append, "decode": _plain_decode, "evict": _plain_evict}[c["kind"]](c, state)


def _own(kind, c, s):
    from native_sparse_attention_triton_b200 import ops

    if kind == "window":
        o = ops.sink_window_attention(s["q"], s["k"], s["v"], s["cu"], c["window"], c["sinks"])
        return (o,) + torch.autograd.grad([o], s["leaves"], [s["do"]]) if c["train"] else (o,)
    if kind == "append":
        after = ops.paged_kv_append(s["kp"], s["vp"], s["table"], s["held"], s["k"], s["v"], s["cu"])
        return s["kp"], s["vp"], after
    if kind == "decode":
        # a decoding loop adds to one buffer step after step; here each pass starts from the same sums
        weights = s["weights"].clone() if c["weights"] else None
        o = ops.paged_attention_decode(s["q"], s["kp"], s["vp"], s["table"], s["lens"], window_size=c["window"] if c["window"] >= 0 else None,
                                       num_sinks=c["sinks"], weights=weights)
        return (o, weights) if c["weights"] else (o,)
    after, weights, kept = ops.paged_kv_evict(s["kp"], s["vp"], s["table"], s["lens"], s["weights"], s["target"], c["budget"], c["sinks"],
                                              c["recent"])
    return s["kp"], s["vp"], after, weights, kept


@torch.no_grad()
def _plain_window(c, s):
    """Blocks of `blk` queries against the keys from `window` before the block to its end, and against every sequence's sinks."""
    hq, hkv, d, left, sinks = c["hq"], c["hkv"], c["d"], c["window"], c["sinks"]
    n, g, cu, seq = s["q"].shape[0], c["hq"] // c["hkv"], s["cu"].long(), s["seq"]
    scale = 1 / math.sqrt(d)
    blk = max(128, left)
    nb = (n + blk - 1) // blk
    at = torch.arange(nb * blk, device=DEVICE)
    row = at.clamp(max=n - 1).view(nb, blk)
    col = torch.arange(nb, device=DEVICE)[:, None] * blk - left + torch.arange(blk + left, device=DEVICE)
    inside, col = (col >= 0) & (col < n), col.clamp(0, n - 1)
    see = (inside[:, None, :] & (at.view(nb, blk) < n)[:, :, None] & (seq[col][:, None, :] == seq[row][:, :, None])
           & (col[:, None, :] <= row[:, :, None]) & (col[:, None, :] >= row[:, :, None] - left))
    sink_pos = torch.arange(sinks, device=DEVICE)
    sink = (cu[:-1, None] + sink_pos).reshape(-1)
    sink_in = (sink_pos < (cu[1:] - cu[:-1])[:, None]).reshape(-1)
    sink = sink.clamp(max=n - 1)
    see_sink = (sink_in & (at.view(nb, blk) < n)[:, :, None] & (seq[sink] == seq[row][:, :, None]) & (sink < row[:, :, None] - left))

    def rows(x):  # [n, hq, d] -> [nb, hkv, blk * g, d]
        return x[row.view(-1)].float().view(nb, blk, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(nb, hkv, blk * g, d)

    def back(x):
        return x.view(nb, hkv, blk, g, d).permute(0, 2, 1, 3, 4).reshape(nb * blk, hq, d)[:n]

    def hide(x, mask, value):
        return x.view(nb, hkv, blk, g, -1).masked_fill_(~mask[:, None, :, None, :], value).view(x.shape)

    q, k, v = rows(s["q"]), s["k"].float(), s["v"].float()
    kw, vw = k[col].permute(0, 2, 1, 3), v[col].permute(0, 2, 1, 3)  # [nb, hkv, cols, d]
    ks, vs = k[sink].permute(1, 0, 2), v[sink].permute(1, 0, 2)      # [hkv, sequences * sinks, d]
    sw = hide((q @ kw.transpose(-1, -2)).mul_(scale), see, -math.inf)
    ss = hide((q @ ks.transpose(-1, -2)).mul_(scale), see_sink, -math.inf)
    top = sw.amax(-1, keepdim=True)
    if sinks:
        top = torch.maximum(top, ss.amax(-1, keepdim=True))
    top = top.clamp(min=-1e30)  # a row that stands for nothing
    pw, ps = sw.sub_(top).exp_(), ss.sub_(top).exp_()
    total = pw.sum(-1, keepdim=True) + ps.sum(-1, keepdim=True)
    total = total.clamp(min=1e-30)
    pw, ps = pw.div_(total), ps.div_(total)
    o = pw @ vw + ps @ vs
    out = back(o).to(s["q"].dtype)
    if not c["train"]:
        return (out,)
    do = rows(s["do"])
    delta = (o * do).sum(-1, keepdim=True)
    dv = torch.zeros(n, hkv, d, device=DEVICE)
    dv.index_add_(0, col.reshape(-1), (pw.transpose(-1, -2) @ do).permute(0, 2, 1, 3).reshape(-1, hkv, d))
    dv.index_add_(0, sink, (ps.transpose(-1, -2) @ do).sum(0).permute(1, 0, 2))
    dw = (do @ vw.transpose(-1, -2)).sub_(delta).mul_(pw).mul_(scale)
    ds = (do @ vs.transpose(-1, -2)).sub_(delta).mul_(ps).mul_(scale)
    dq = dw @ kw + ds @ ks
    dk = torch.zeros(n, hkv, d, device=DEVICE)
    dk.index_add_(0, col.reshape(-1), (dw.transpose(-1, -2) @ q).permute(0, 2, 1, 3).reshape(-1, hkv, d))
    dk.index_add_(0, sink, (ds.transpose(-1, -2) @ q).sum(0).permute(1, 0, 2))
    t = s["q"].dtype
    return out, back(dq).to(t), dk.to(t), dv.to(t)


def _plain_append(c, s):
    new = torch.ones_like(s["held"]) if s["cu"] is None else s["cu"][1:] - s["cu"][:-1]
    first = torch.cumsum(new, 0) - new
    pos = s["held"][s["seq"]] + torch.arange(s["k"].shape[0], device=DEVICE) - first[s["seq"]]
    page, slot = s["table"][s["seq"], pos // c["page"]].long(), pos % c["page"]
    s["kp"][page, slot] = s["k"]
    s["vp"][page, slot] = s["v"]
    return s["kp"], s["vp"], s["held"] + new.int()


def _plain_decode(c, s):
    b, hkv, d = s["q"].shape[0], c["hkv"], c["d"]
    g = c["hq"] // hkv
    table = s["table"].long()
    cap = table.shape[1] * c["page"]
    at, n = torch.arange(cap, device=DEVICE), s["lens"][:, None]
    see = at < n
    if c["window"] >= 0:
        see = see & ((at >= n - 1 - c["window"]) | (at < c["sinks"]))
    see = see[:, None, None, :]
    k = s["kp"][table].view(b, cap, hkv, d).permute(0, 2, 3, 1).float()
    x = (s["q"].float().view(b, hkv, g, d) @ k).mul_(1 / math.sqrt(d)).masked_fill_(~see, -math.inf)
    del k
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p = x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30))
    o = (p @ s["vp"][table].view(b, cap, hkv, d).permute(0, 2, 1, 3).float()).view(b, c["hq"], d).to(s["q"].dtype)
    return (o, s["weights"] + p.sum(2)) if c["weights"] else (o,)


def _plain_evict(c, s):
    b, hkv, cap = s["weights"].shape
    n, at = s["lens"][:, None, None], torch.arange(cap, device=DEVICE)
    forced = (at < c["sinks"]) | (at >= n - c["recent"])
    rank = torch.where(at >= n, -math.inf, torch.where(forced, math.inf, s["weights"]))
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    kept = torch.where(kept < n, kept, cap).sort(-1).values              # ascending, the empty ones last
    if kept.shape[-1] < c["budget"]:
        kept = torch.nn.functional.pad(kept, (0, c["budget"] - kept.shape[-1]), value=cap)
    there = kept < cap
    seq, head, to = there.nonzero(as_tuple=True)
    src = kept[there]
    from_page, to_page = s["table"][seq, src // c["page"]].long(), s["target"][seq, to // c["page"]].long()
    s["kp"][to_page, to % c["page"], head] = s["kp"][from_page, src % c["page"], head]
    s["vp"][to_page, to % c["page"], head] = s["vp"][from_page, src % c["page"], head]
    weights = torch.zeros_like(s["weights"])
    weights[seq, head, to] = s["weights"][seq, head, src]
    return s["kp"], s["vp"], s["lens"].clamp(max=c["budget"]), weights, torch.where(there, kept, -1).int()


# ------------------------------------------------------------------------------------------------------------- definitions
def exact(case, seed):
    """The operators' definitions, sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"window": _exact_window, "append": _exact_append, "decode": _exact_decode, "evict": _exact_evict}[case["kind"]](case, s)


def _exact_window(c, s):
    g, scale = c["hq"] // c["hkv"], c["d"] ** -0.5
    out = [torch.zeros(x.shape, dtype=torch.float64, device=DEVICE) for x in (s["q"], s["q"], s["k"], s["v"])]
    start = 0
    for n in _ints(c["lens"]):
        i, j = torch.arange(n, device=DEVICE)[:, None], torch.arange(n, device=DEVICE)[None, :]
        see = (j <= i) & ((i - j <= c["window"]) | (j < c["sinks"]))
        part = slice(start, start + n)
        for h in range(c["hq"]):
            q, k, v = s["q"][part, h].double(), s["k"][part, h // g].double(), s["v"][part, h // g].double()
            p = torch.softmax((q @ k.T * scale).masked_fill(~see, -math.inf), dim=1)
            out[0][part, h] = o = p @ v
            if c["train"]:
                do = s["do"][part, h].double()
                t = p * (do @ v.T - (o * do).sum(1, keepdim=True)) * scale
                out[1][part, h] = t @ k
                out[2][part, h // g] += t.T @ q
                out[3][part, h // g] += p.T @ do
        start += n
    return tuple(out) if c["train"] else (out[0],)


def _exact_append(c, s):
    kp, vp, table, start = s["kp"].double(), s["vp"].double(), s["table"].tolist(), 0
    for b, (held, new) in enumerate(zip(_ints(c["lens"]), _ints(c["new"]))):
        at = 0
        while at < new:  # page by page
            page, slot = table[b][(held + at) // c["page"]], (held + at) % c["page"]
            take = min(new - at, c["page"] - slot)
            kp[page, slot:slot + take] = s["k"][start + at:start + at + take].double()
            vp[page, slot:slot + take] = s["v"][start + at:start + at + take].double()
            at += take
        start += new
    return kp, vp, None


def _rows_of(pages, table, n, page):
    """The first n rows of a sequence, in order."""
    return pages[table[:(n + page - 1) // page].long()].flatten(0, 1)[:n]


def _exact_decode(c, s):
    g, o = c["hq"] // c["hkv"], torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    weights = s["weights"].double() if c["weights"] else None
    for b, n in enumerate(_ints(c["lens"])):
        k, v = _rows_of(s["kp"], s["table"][b], n, c["page"]), _rows_of(s["vp"], s["table"][b], n, c["page"])
        rows = torch.arange(n, device=DEVICE)
        if c["window"] >= 0:
            rows = rows[(rows < c["sinks"]) | (rows + c["window"] >= n - 1)]
        for h in range(c["hkv"]):
            p = torch.softmax(s["q"][b, h * g:h * g + g].double() @ k[rows, h].double().T / c["d"] ** 0.5, dim=1)
            o[b, h * g:h * g + g] = p @ v[rows, h].double()
            if c["weights"]:
                weights[b, h, rows] += p.sum(0)
    return (o, weights) if c["weights"] else (o,)


def _exact_evict(c, s):
    kp, vp = s["kp"].double(), s["vp"].double()
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_ints(c["lens"])):
        k, v = _rows_of(s["kp"], s["table"][b], n, c["page"]), _rows_of(s["vp"], s["table"][b], n, c["page"])
        m = min(n, c["budget"])
        to = torch.arange(m, device=DEVICE)
        page, slot = s["target"][b].long()[to // c["page"]], to % c["page"]
        for h in range(c["hkv"]):
            w = s["weights"][b, h, :n].double()
            if n > m:
                middle = range(c["sinks"], n - c["recent"])
                best = torch.sort(-w[middle.start:middle.stop], stable=True).indices[:m - c["sinks"] - c["recent"]] + middle.start
                rows = torch.cat([torch.arange(c["sinks"], device=DEVICE), best.sort().values, torch.arange(n - c["recent"], n, device=DEVICE)])
            else:
                rows = to
            kp[page, slot, h], vp[page, slot, h], weights[b, h, :m] = k[rows, h].double(), v[rows, h].double(), w[rows]
    return kp, vp, None, weights, None


# ------------------------------------------------------------------------------------------------------------------- work
def _seen(n, c):
    """Keys that the last of n tokens sees."""
    return n if c["window"] < 0 else min(n, c["window"] + 1) + max(0, min(c["sinks"], n - c["window"] - 1))


def work(case):
    c, lens = case, _ints(case["lens"])
    hkv, d = c["hkv"], c["d"]
    row = 2 * hkv * d  # bytes of a key (or value) row
    if c["kind"] == "window":
        pairs = sum(_seen(t, c) for n in lens for t in range(1, n + 1))
        q, kv = 2 * sum(lens) * c["hq"] * d, sum(lens) * row
        # q, k, v in and o out; with training the upstream gradient in and the three gradients out
        return {"bytes": 2 * q + 2 * kv + (2 * q + 2 * kv if c["train"] else 0), "flops": (14 if c["train"] else 4) * d * c["hq"] * pairs}
    if c["kind"] == "append":
        return {"bytes": 2 * 2 * sum(_ints(c["new"])) * row, "flops": 0}
    if c["kind"] == "decode":
        rows = sum(_seen(n, c) for n in lens)
        return {"bytes": 2 * rows * row + 2 * 2 * len(lens) * c["hq"] * d + (8 * hkv * rows if c["weights"] else 0), "flops": 4 * rows * c["hq"] * d}
    rows = sum(min(n, c["budget"]) for n in lens)
    # K and V rows in and out; the sums of all rows in, those of the kept ones out, their numbers out
    return {"bytes": 2 * 2 * rows * row + 4 * hkv * (sum(lens) + 2 * rows), "flops": 0}
