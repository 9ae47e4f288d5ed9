"""64-bit references of the sliding window with sinks and of the paged operators, and the bounds that their roundings give.

A kernel rounds a result to its type: at most h = eps / 2 of it.  sink_window_attention also rounds the probabilities P and, backward, dS to
16 bits before they enter a product, h of each of them, and takes a share of the exponentials from a cubic of relative error 7.5e-5.
SLACK stands for that cubic, the exponential unit (2^-22) and the fp32 sums: of a logit's 128 products, 2^-24 each of sum |q k| scale, below
2e-5 for the inputs here, and of the sums over keys, which grow with their number, 2^-24 sqrt(n) and below 2e-5 for up to 10^5 terms.

A rounding is at most h of the value only where that is a normal number.  Below tiny, the smallest one (2^-14 in fp16), numbers are tiny * eps apart,
so there a rounding is up to u = tiny * eps / 2 (2^-25) whatever the value.  That goes for a result, for each dS, and for each P: 2^(x - m)
with m no larger than the row's maximum, so that their sum is at least 1 and u of each is no more than u after the division; backward P is
normalised already.  (fp16, no sinks, 431 keys: a gradient of -2.876e-7 comes as -2.980e-7, its neighbour, 1.0e-8 < 2^-25 = 3.0e-8 off.)
"""
import math

import torch

SLACK = 3e-4
DECODE_SLACK = 6e-5  # no cubic, P as two 16-bit numbers (2^-17)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least_step(dtype):
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def window_mask(n, window, sinks, device):
    i, j = torch.arange(n, device=device)[:, None], torch.arange(n, device=device)[None, :]
    return (j <= i) & ((i - j <= window) | (j < sinks))


def sink_window(q, k, v, lens, window, sinks, do=None, scale=None):
    """(values, bounds), each [o] or [o, dq, dk, dv] in 64 bits.  Rows behind the last sequence are zero."""
    g, d = q.shape[1] // k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    h, u = half_step(q.dtype), least_step(q.dtype)
    n_out = 1 if do is None else 4
    val = [torch.zeros(x.shape, dtype=torch.float64, device=q.device) for x in (q, q, k, v)[:n_out]]
    tol = [torch.zeros_like(x) for x in val]
    start = 0
    for n in lens:
        part = slice(start, start + n)
        see = window_mask(n, window, sinks, q.device)
        for head in range(q.shape[1] if n else 0):
            kv = head // g
            qh, kh, vh = q[part, head].double(), k[part, kv].double(), v[part, kv].double()
            p = torch.softmax((qh @ kh.T * scale).masked_fill(~see, -math.inf), 1)
            o, mass = p @ vh, p @ vh.abs()
            val[0][part, head] = o
            o_err = h * o.abs() + u + (h + SLACK) * mass + u * (see.double() @ vh.abs())
            tol[0][part, head] = o_err
            if do is None:
                continue
            g_ = do[part, head].double()
            dp, delta = g_ @ vh.T, (o * g_).sum(1, keepdim=True)
            ds = p * (dp - delta) * scale
            # of dS: its rounding, that of o in delta (o is kept as two 16-bit numbers; one rounding of each P in it is allowed for, which the
            # two parts of P that a forward has for a backward pass stay far below), and the
            # 32-bit arithmetic of its parts
            o_kept = o_err - (h - h * h) * o.abs()
            err = h * ds.abs() + u * see + p * scale * (o_kept * g_.abs()).sum(1, keepdim=True) + SLACK * p * scale * (g_.abs() @ vh.abs().T + delta.abs())
            val[1][part, head] = ds @ kh
            tol[1][part, head] = err @ kh.abs()
            val[2][part, kv] += ds.T @ qh
            tol[2][part, kv] += err.T @ qh.abs()
            val[3][part, kv] += p.T @ g_
            tol[3][part, kv] += ((h + SLACK) * p + u * see).T @ g_.abs()
        start += n
    for x, t in list(zip(val, tol))[1:]:
        t += h * x.abs() * (1 + h) + u  # the result's own rounding
    return val, tol


def rows_of(pages, table_row, n):
    """The first n rows of a sequence, in order: [n, heads, d]."""
    page = pages.shape[1]
    return pages[table_row[:(n + page - 1) // page].long()].flatten(0, 1)[:n]


def seen_rows(n, window, sinks, device):
    j = torch.arange(n, device=device)
    return j if window is None else j[(n - 1 - j <= window) | (j < sinks)]


def paged_decode(q, kp, vp, table, lens, window=None, sinks=0, scale=None):
    """(o, its bound, [(rows, weights [heads, rows])] per sequence) in 64 bits."""
    hkv, d = kp.shape[2], kp.shape[3]
    g = q.shape[1] // hkv
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol, weights = torch.zeros_like(o), []
    for b, n in enumerate(lens):
        rows = seen_rows(n, window, sinks, q.device)
        if n == 0:
            weights.append((rows, torch.zeros(hkv, 0, dtype=torch.float64, device=q.device)))
            continue
        k, v = rows_of(kp, table[b], n)[rows].double(), rows_of(vp, table[b], n)[rows].double()
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[b].double().view(hkv, g, d), k) * scale, -1)
        o[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(q.shape[1], d)
        mass = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(q.shape[1], d)
        # (the two numbers of a P are 2^-25 apart from it at most too)
        tol[b] = half_step(q.dtype) * o[b].abs() + least_step(q.dtype) + DECODE_SLACK * mass
        weights.append((rows, p.sum(1)))
    return o, tol, weights


def evict_rows(w, n, budget, sinks, recent):
    """The rows kept of a sequence of n rows with weights w [n]: ascending list, from the definition."""
    if n <= budget:
        return list(range(n))
    w = [float("-inf") if math.isnan(x) else x for x in w.tolist()]
    between = sorted(range(sinks, n - recent), key=lambda j: (-w[j], j))[:budget - sinks - recent]
    return list(range(sinks)) + sorted(between) + list(range(n - recent, n))


def assert_within(got, value, bound, name=""):
    got = got.double()
    assert got.shape == value.shape
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got - value).abs() - bound) / (bound + 1e-30)
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0, f"{name}: {1 + worst:.3f} of the bound, value {value.flatten()[over.argmax()]:.4g}, got {got.flatten()[over.argmax()]:.4g}"
