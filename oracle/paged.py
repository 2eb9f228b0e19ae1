"""Paged KV cache in 64 bits: what an append leaves and what attention to the pages returns.

Written row by row from the definition, on torch tensors of any device; caches are given and
returned in [pages, page_size, heads, d] order.
"""

import math

import torch

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


def rotate(x, pos, cos, sin, rotary, interleaved):
    """x [heads, d] float64, rotated by row `pos` of the tables."""
    y = x.clone()
    c, s = cos[pos].double(), sin[pos].double()
    first = torch.arange(rotary // 2, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else rotary // 2)
    y[:, first] = x[:, first] * c - x[:, second] * s
    y[:, second] = x[:, second] * c + x[:, first] * s
    return y


def append_rows(x, table, lens, starts, page_size, num_pages, turn):
    """{(page, head-major row): values} of the rows that an append of packed x [total, heads, d]
    stores: a dict (page, slot) -> [heads, d] float64, and {page: first new slot}."""
    rows, first = {}, {}
    for b, n in enumerate(lens):
        for i in range(starts[b + 1] - starts[b]):
            pos = max(n, 0) + i
            if pos >= table.shape[1] * page_size:
                break
            page, slot = int(table[b, pos // page_size]), pos % page_size
            if not 0 <= page < num_pages:
                continue
            rows[page, slot] = turn(x[starts[b] + i].double(), pos)
            first[page] = min(first.get(page, slot), slot)
    return rows, first


def attend(q, k_cache, v_cache, table, lens, starts, scale, causal, k_scale=None, v_scale=None):
    """o [total, Hq, d] and lse [total, Hq] in float64, and, per output element, the sums over the
    seen rows of p |v| (`mass`) and of |v| in units of the largest value scale (`spread`), from
    which an error bound follows; `qk` is the largest sum of |q k| |scale|."""
    total, hq, d = q.shape
    num_pages, page_size, hkv, _ = k_cache.shape
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass, spread = torch.zeros_like(o), torch.zeros_like(o)
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64, device=q.device)
    qk = 0.0
    for b, n in enumerate(lens):
        t0, t1 = starts[b], starts[b + 1]
        n = min(max(n, 0), table.shape[1] * page_size)
        if t0 == t1 or n == 0:
            continue
        pages = table[b, :-(-n // page_size)].long()
        good = ((pages >= 0) & (pages < num_pages)).repeat_interleave(page_size)[:n]
        pages = pages.clamp(0, num_pages - 1)
        k, v = k_cache[pages].double(), v_cache[pages].double()
        unit = torch.ones((len(pages), hkv), dtype=torch.float64, device=q.device)
        if k_scale is not None:
            k = k * k_scale[pages].double()[:, None, :, None]
            unit = v_scale[pages].double()
            v = v * unit[:, None, :, None]
        k, v = (t.reshape(-1, hkv, d)[:n][good] for t in (k, v))
        unit = unit.repeat_interleave(page_size, 0)[:n][good]
        at = torch.arange(n, device=q.device)[good]
        i = torch.arange(t1 - t0, device=q.device)[:, None]
        seen = at[None] <= n - (t1 - t0) + i if causal else torch.ones((t1 - t0, len(at)), dtype=torch.bool, device=q.device)
        for h in range(hq):
            g = h // (hq // hkv)
            qh = q[t0:t1, h].double()
            x = (qh @ k[:, g].T * scale).masked_fill(~seen, -math.inf)
            qk = max(qk, float(((qh.abs() @ k[:, g].abs().T) * abs(scale)).max()) if len(at) else 0.0)
            some = seen.any(-1)
            p = torch.where(some[:, None], torch.softmax(x, -1), torch.zeros_like(x))
            o[t0:t1, h] = p @ v[:, g]
            lse[t0:t1, h] = torch.logsumexp(x, -1)
            mass[t0:t1, h] = p @ v[:, g].abs()
            if len(at):
                spread[t0:t1, h] = seen.double() @ (v[:, g].abs() * (unit[:, g].max() / unit[:, g])[:, None])
    return o, lse, mass, spread, qk
