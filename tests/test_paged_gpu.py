"""Paged KV cache on the GPU: rotation and append, attention to the pages, and both in a serving
loop, against the 64-bit definition (oracle/paged.py).

Tolerances, u = torch.finfo(dtype).eps / 2 (half a step of the 16-bit type):
* a stored row: its rotation in fp32 is off by at most 3 roundings of |x1| + |x2|, then one
  rounding: half a step of the cache's type (e4m3: 2^-4 of the value, or 2^-10 units of the scale);
* attention: the probabilities are rounded to the 16-bit type (u of each; fp16 also 2^-25 of the
  largest where they fall below its normal numbers) and the result once more (u); scores are off
  by e = d 2^-24 sum|q k| at most, which moves every probability and their sum by e; sums over n
  rows by n 2^-24; the hardware's exp2 and the rescaling by 2^-20.
"""

import math

import pytest
import torch

from oracle import paged as orc

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def starts_of(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


class Pool:
    """Pages with content, page tables and scales for sequences of up to `capacity` rows."""

    def __init__(self, seqs, pages_per_seq, page, hkv, d, cache, dtype=torch.float16, layout="bshd", seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.page, self.hkv, self.d, self.layout, self.dtype = page, hkv, d, layout, dtype
        self.pages = seqs * pages_per_seq + spare
        self.table = torch.randperm(self.pages, generator=g)[:seqs * pages_per_seq].view(seqs, pages_per_seq).int().cuda()
        shape = (self.pages, page, hkv, d)
        self.k_scale = self.v_scale = None
        kind = FP8 if cache == "fp8" else dtype
        values = [torch.randn(shape, generator=g), torch.randn(shape, generator=g)]
        if kind == FP8:
            self.k_scale, self.v_scale = (torch.exp2(torch.randint(-9, -4, (self.pages, hkv), generator=g).float()).cuda()
                                          for _ in range(2))
            values = [(x * 100).clamp(-448, 448) for x in values]
        caches = [x.to(kind) for x in values]
        if layout == "bhsd":
            caches = [x.transpose(1, 2).contiguous() for x in caches]
        self.k_cache, self.v_cache = (x.cuda() for x in caches)

    def rows(self, cache):
        return cache if self.layout == "bshd" else cache.transpose(1, 2)

    def append(self, k, v, lens, **kw):
        from flash_attn_legacy import paged_kvcache_append
        lens = torch.tensor(lens, dtype=torch.int32).cuda() if isinstance(lens, list) else lens
        return paged_kvcache_append(k, v, self.k_cache, self.v_cache, self.table, lens, k_scale=self.k_scale,
                                    v_scale=self.v_scale, cache_layout=self.layout, **kw)

    def attend(self, q, lens, **kw):
        from flash_attn_legacy import flash_attn_with_paged_kvcache
        lens = torch.tensor(lens, dtype=torch.int32).cuda() if isinstance(lens, list) else lens
        return flash_attn_with_paged_kvcache(q, self.k_cache, self.v_cache, self.table, lens, k_scale=self.k_scale,
                                             v_scale=self.v_scale, cache_layout=self.layout, **kw)


def randn(shape, seed, dtype=torch.float16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def tiny(dtype):
    """The smallest subnormal number"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def same(a, b):
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.contiguous().view(bits), b.contiguous().view(bits))


def check_append(pool, k, v, lens, new, before, cos=None, sin=None, rotary=0, interleaved=False):
    """The caches and scales after an append of packed k, v, given what they were `before`."""
    starts = starts_of(new)
    table = pool.table.cpu()
    for name, x, turned in (("k", k, rotary > 0), ("v", v, False)):
        turn = (lambda y, p: orc.rotate(y, p, cos, sin, rotary, interleaved)) if turned else lambda y, p: y
        want, first = orc.append_rows(x, table, lens, starts, pool.page, pool.pages, turn)
        got, old = pool.rows(getattr(pool, name + "_cache")), pool.rows(before[name + "_cache"])
        slack = 3 * 2.0 ** -24 * 2 * (float(x.double().abs().max()) if x.numel() else 0.0) if turned else 0.0
        untouched = torch.ones(got.shape[:2], dtype=torch.bool)
        for page, slot in want:
            untouched[page, slot] = False
        if pool.k_scale is None:
            u = torch.finfo(x.dtype).eps / 2
            for (page, slot), y in want.items():
                err = (got[page, slot].double() - y).abs()
                assert bool((err <= u * y.abs() + 2 * slack + tiny(x.dtype)).all()), (name, page, slot, float(err.max()))
        else:
            s_new, s_old = (t.double() for t in (getattr(pool, name + "_scale"), before[name + "_scale"]))
            for page, slot0 in first.items():
                fresh = torch.stack([y for (p, _), y in want.items() if p == page])       # [rows, heads, d]
                amax = fresh.abs().amax((0, 2))
                s = s_new[page]
                floor = s_old[page] if slot0 else torch.full_like(s, orc.MIN_SCALE)
                assert bool((torch.frexp(s)[0] == 0.5).all()) and bool((s >= floor).all())
                assert bool((448 * s >= amax * (1 - 2.0 ** -22)).all()), (name, page)
                assert bool(((s == floor) | (224 * s < amax * (1 + 2.0 ** -22))).all()), (name, page)
                untouched[page, :slot0] = False
                a = got[page, :slot0].double() * s[:, None]
                y = old[page, :slot0].double() * s_old[page][:, None]
                kept = (s == s_old[page])[None, :, None]
                bound = torch.maximum(y.abs() * 2.0 ** -4, s[:, None] * 2.0 ** -10)
                assert bool(torch.where(kept, a == y, (a - y).abs() <= bound).all()), (name, page)
            for (page, slot), y in want.items():
                s = s_new[page][:, None]
                err = (got[page, slot].double() * s - y).abs()
                bound = torch.maximum(y.abs() * 2.0 ** -4, s * 2.0 ** -10) + 2 * slack
                assert bool((err <= bound).all()), (name, page, slot, float((err / bound).max()))
            rest = torch.ones(pool.pages, dtype=torch.bool)
            rest[list(first)] = False
            assert same(getattr(pool, name + "_scale")[rest.cuda()], before[name + "_scale"][rest.cuda()])
        mask = untouched.cuda()
        raw = (lambda t: t.view(torch.uint8)) if pool.k_scale is not None else (lambda t: t.view(torch.int16))
        assert torch.equal(raw(got.contiguous())[mask], raw(old.contiguous())[mask]), name


def snapshot(pool):
    return {n: getattr(pool, n).clone() for n in ("k_cache", "v_cache", "k_scale", "v_scale") if getattr(pool, n) is not None}


def check_attend(pool, q, lens, new, got, causal=True, scale=None, table=None):
    """o and lse of packed q [total, Hq, d] (or [B, n, Hq, d])."""
    o, lse = (t.reshape(-1, *t.shape[q.dim() - 2:]) for t in got)
    flat = q.reshape(-1, *q.shape[-2:])
    d = q.shape[-1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    ro, rl, mass, spread, qk = orc.attend(flat, pool.rows(pool.k_cache), pool.rows(pool.v_cache), pool.table, lens,
                                          starts_of(new), scale, causal, pool.k_scale, pool.v_scale)
    u = torch.finfo(q.dtype).eps / 2
    n = max([0, *lens])
    e = d * 2.0 ** -24 * qk
    tol = mass * (2 * u + 2 * e + (n + 64) * 2.0 ** -24 + 2.0 ** -20) + tiny(q.dtype)
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * spread
    err = (o.double() - ro).abs()
    assert bool((err <= tol).all()), f"o: {float((err / tol).max()):.3g} of the tolerance"
    none = torch.isneginf(rl)
    assert torch.equal(torch.isneginf(lse), none)
    off = torch.where(none, torch.zeros_like(rl), (lse.double() - rl).abs())
    lse_tol = e + (n + 64) * 2.0 ** -24 + 2.0 ** -20 * (1 + rl.abs().nan_to_num(posinf=0))
    assert bool((off <= lse_tol).all()), f"lse: {float((off / lse_tol).max()):.3g} of the tolerance"
    assert bool((o[none] == 0).all())


# ---- append ----------------------------------------------------------------------------------

APPENDS = [
    # d, page, hkv, hq, layout, dtype, rotary, interleaved, lens, new (packed when they differ)
    (128, 64, 2, 8, "bshd", torch.bfloat16, 128, False, [0, 5, 63, 64, 100], [1, 1, 1, 1, 1]),
    (128, 64, 2, 4, "bhsd", torch.float16, 64, False, [0, 17, 64, 1], [130, 0, 1, 63]),
    (64, 16, 3, 3, "bshd", torch.float16, 64, True, [15, 16, 31, 0], [2, 17, 1, 40]),
    (32, 48, 1, 8, "bhsd", torch.bfloat16, 16, True, [47, 3], [5, 200]),
    (96, 32, 2, 4, "bshd", torch.float16, 96, False, [31, 0, 8], [33, 33, 33]),
    (256, 128, 2, 2, "bshd", torch.bfloat16, 256, False, [100, 0], [29, 300]),
    (128, 256, 1, 1, "bhsd", torch.float16, 128, True, [255, 0], [2, 256]),
    (64, 64, 2, 6, "bshd", torch.bfloat16, 0, False, [7, 120], [64, 9]),
]


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"d{c[0]}p{c[1]}{c[4]}r{c[6]}{'i' if c[7] else ''}")
def test_append(case, cache):
    from flash_attn_legacy import rotary_cos_sin
    d, page, hkv, hq, layout, dtype, rotary, inter, lens, new = case
    per = max(-(-(a + n) // page) for a, n in zip(lens, new)) + 1
    pool = Pool(len(lens), per, page, hkv, d, cache, dtype, layout, seed=d + page)
    total = sum(new)
    k, v, q = randn((total, hkv, d), 1, dtype, 3.0), randn((total, hkv, d), 2, dtype), randn((total, hq, d), 3, dtype)
    k[..., 1] *= 20
    cos, sin = rotary_cos_sin(per * page, rotary, device="cuda") if rotary else (None, None)
    before = snapshot(pool)
    kw = dict(rotary_cos=cos, rotary_sin=sin, rotary_interleaved=inter)
    if len(set(new)) == 1:
        four = lambda x: x.view(len(new), new[0], *x.shape[1:])
        rq = pool.append(four(k), four(v), lens, q=four(q), **kw).view(q.shape)
    else:
        cu = torch.tensor(starts_of(new), dtype=torch.int32).cuda()
        rq = pool.append(k, v, lens, q=q, cu_seqlens=cu, max_seqlen=max(new), **kw)
    check_append(pool, k, v, lens, new, before, cos, sin, rotary, inter)
    u = torch.finfo(dtype).eps / 2
    for b, t0 in enumerate(starts_of(new)[:-1]):
        for i in range(new[b]):
            y = q[t0 + i].double()
            if rotary:
                y = orc.rotate(y, lens[b] + i, cos, sin, rotary, inter)
            err = (rq[t0 + i].double() - y).abs()
            assert bool((err <= u * y.abs() + 2.0 ** -20).all()), (b, i, float(err.max()))


@pytest.mark.parametrize("cache", ["fp8", "same"])
def test_append_hint_shorter_than_the_sequences(cache):
    """max_seqlen only sizes the grid."""
    pool, other = (Pool(2, 5, 16, 2, 64, cache, seed=4) for _ in range(2))
    new, lens = [70, 33], [3, 20]
    k, v = randn((103, 2, 64), 1), randn((103, 2, 64), 2)
    cu = torch.tensor(starts_of(new), dtype=torch.int32).cuda()
    pool.append(k, v, lens, cu_seqlens=cu, max_seqlen=1)
    other.append(k, v, lens, cu_seqlens=cu, max_seqlen=70)
    assert same(pool.k_cache, other.k_cache) and same(pool.v_cache, other.v_cache)
    check_append(pool, k, v, lens, new, snapshot(Pool(2, 5, 16, 2, 64, cache, seed=4)))


@pytest.mark.parametrize("page", [16, 64])
def test_scales_grow_with_later_tokens(page):
    """Tokens that grow and shrink, one by one: the scale only grows while a page fills, the older
    rows stay within a rounding of each growth, and a page's first row starts afresh."""
    pool = Pool(1, 3, page, 2, 64, "fp8", torch.bfloat16, seed=1)
    size = torch.tensor([2.0 ** ((i * 5) % 13 - 6) for i in range(2 * page + 3)])
    k = (torch.randn(len(size), 2, 64, generator=torch.Generator().manual_seed(3)) * size[:, None, None]).bfloat16().cuda()
    for i in range(len(size)):
        before = snapshot(pool)
        pool.append(k[i][None, None], k[i][None, None], [i])
        check_append(pool, k[i:i + 1], k[i:i + 1], [i], [1], before)


def test_append_special_values():
    """Zeros, infinities, NaN and values at the ends of bfloat16's range."""
    pool = Pool(6, 1, 16, 1, 32, "fp8", torch.bfloat16, seed=2)
    k = torch.ones((6, 3, 1, 32), dtype=torch.bfloat16)
    k[0] = 0
    k[1, 1, 0, 5], k[1, 2, 0, 6] = math.inf, -math.inf
    k[2, 0, 0, 3] = math.nan
    k[3] *= 3.0e38
    k[4] *= 1.0e-38
    k[5, 0, 0, 0] = 448
    k = k.cuda()
    pool.append(k, k, [0] * 6)
    page = pool.table[:, 0].long()
    code, scale = pool.k_cache[page].float()[:, :3, 0], pool.k_scale[page, 0].double()
    assert scale[0] == 2.0 ** -126 and bool((code[0] == 0).all())
    assert scale[1] == 2.0 ** -8 and code[1, 1, 5] == 448 and code[1, 2, 6] == -448 and bool((code[1, 0] == 256).all())
    assert scale[2] == 2.0 ** -8 and torch.isnan(code[2, 0, 3]) and int(torch.isnan(code[2]).sum()) == 1
    assert scale[3] == 2.0 ** 120 and bool((code[3] == 224).all())      # 3e38 in bfloat16: 226 * 2^120, steps of 16
    assert scale[4] == 2.0 ** -126 and bool((code[4] == 0.875).all())   # 1e-38 in bfloat16: 0.8516 * 2^-126, steps of 1/16
    assert scale[5] == 1 and code[5, 0, 0] == 448
    # an infinity behind ordinary rows leaves the page's scale and the rows
    more = torch.full((6, 1, 1, 32), math.inf, dtype=torch.bfloat16).cuda()
    before = snapshot(pool)
    pool.append(more, more, [3] * 6)
    assert torch.equal(pool.k_scale, before["k_scale"]) and bool((pool.k_cache[page].float()[:, 3] == 448).all())


@pytest.mark.parametrize("cache", ["fp8", "same"])
def test_append_drops_what_has_no_page(cache):
    """Page ids outside the pool, rows past the table and negative lengths: nothing else changes."""
    pool = Pool(4, 3, 16, 2, 64, cache, seed=5)
    pool.table[0, 1] = -1
    pool.table[1, 0] = pool.pages
    pool.table[2, 2] = 2 ** 31 - 1
    lens, new = [0, 10, 20, 30], [40, 40, 40, 40]
    k, v, q = randn((160, 2, 64), 1), randn((160, 2, 64), 2), randn((160, 4, 64), 3)
    before = snapshot(pool)
    four = lambda x: x.view(4, 40, *x.shape[1:])
    rq = pool.append(four(k), four(v), lens, q=four(q))
    check_append(pool, k, v, lens, new, before)
    for b, n in enumerate(lens):       # not rotated: the rows themselves, and zeros past the table's 48
        fits = min(40, 48 - n)
        assert torch.equal(rq[b, :fits], four(q)[b, :fits]) and bool((rq[b, fits:] == 0).all())
    before = snapshot(pool)
    pool.append(four(k), four(v), [-5, 2 ** 31 - 1, 48, -(2 ** 31)])
    check_append(pool, k, v, [0, 48, 48, 0], new, before)


def test_append_packed_rows_outside_every_sequence():
    pool = Pool(3, 2, 16, 1, 64, "fp8", seed=6)
    k, v, q = randn((40, 1, 64), 1), randn((40, 1, 64), 2), randn((40, 2, 64), 3)
    cu = torch.tensor([4, 9, 9, 30], dtype=torch.int32).cuda()
    before = snapshot(pool)
    rq = pool.append(k, v, [1, 2, 3], q=q, cu_seqlens=cu, max_seqlen=21)
    check_append(pool, k[4:30], v[4:30], [1, 2, 3], [5, 0, 21], before)
    assert torch.equal(rq[4:30], q[4:30]) and bool((rq[:4] == 0).all()) and bool((rq[30:] == 0).all())


def test_append_strided_operands():
    """k and v as halves of one projection, caches as halves of one pool, scales and tables as
    slices, heads of q through a transpose."""
    pool = Pool(2, 2, 32, 2, 64, "fp8", seed=7)
    both = torch.stack([pool.k_cache, pool.v_cache], 1)              # [pages, 2, page, heads, d]
    scales = torch.stack([pool.k_scale, pool.v_scale], -1)           # [pages, heads, 2]
    table = torch.zeros((2, 7), dtype=torch.int32).cuda()
    table[:, 2:4] = pool.table
    before = snapshot(pool)
    pool.k_cache, pool.v_cache = both[:, 0], both[:, 1]
    pool.k_scale, pool.v_scale = scales[..., 0], scales[..., 1]
    pool.table = table[:, 2:4]
    kv = randn((2, 9, 2, 2, 64), 1)
    q = randn((2, 4, 9, 64), 2).transpose(1, 2)
    rq = pool.append(kv[:, :, 0], kv[:, :, 1], [30, 0], q=q)
    check_append(pool, kv[:, :, 0].reshape(18, 2, 64), kv[:, :, 1].reshape(18, 2, 64), [30, 0], [9, 9], before)
    assert torch.equal(rq, q)
    got = pool.attend(q, [39, 9], return_softmax_lse=True)
    check_attend(pool, q.contiguous(), [39, 9], [9, 9], got)


# ---- attention -------------------------------------------------------------------------------

ATTENDS = [
    # d, page, hkv, hq, layout, dtype, lens (with the new rows), new
    (128, 64, 2, 8, "bshd", torch.bfloat16, [1, 64, 65, 700], [1, 1, 1, 1]),
    (128, 16, 8, 32, "bshd", torch.float16, [333, 2000], [1, 1]),
    (64, 16, 12, 12, "bhsd", torch.float16, [5, 129, 1030], [1, 1, 1]),
    (32, 32, 1, 8, "bshd", torch.bfloat16, [31, 300], [1, 1]),
    (96, 48, 2, 8, "bhsd", torch.float16, [49, 500], [1, 1]),
    (256, 128, 2, 4, "bshd", torch.bfloat16, [130, 600], [1, 1]),
    (128, 64, 1, 40, "bshd", torch.bfloat16, [90, 257], [1, 1]),
    (128, 64, 2, 14, "bhsd", torch.float16, [70, 300], [5, 5]),
    (64, 64, 2, 8, "bshd", torch.bfloat16, [40, 333, 64], [17, 17, 17]),
    (128, 32, 2, 8, "bshd", torch.float16, [130, 257, 9, 64], [130, 1, 9, 33]),
    (96, 16, 1, 4, "bshd", torch.bfloat16, [200, 40], [100, 40]),
    (256, 64, 1, 2, "bhsd", torch.float16, [150, 333], [70, 129]),
    (32, 256, 2, 2, "bhsd", torch.float16, [300, 70], [257, 3]),
    (64, 128, 1, 3, "bshd", torch.float16, [700, 129], [301, 129]),
]


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: f"d{c[0]}p{c[1]}h{c[3]}-{c[2]}{c[4]}n{max(c[7])}")
def test_attend(case, causal, cache):
    d, page, hkv, hq, layout, dtype, lens, new = case
    pool = Pool(len(lens), -(-max(lens) // page), page, hkv, d, cache, dtype, layout, seed=d + hq)
    q = randn((sum(new), hq, d), 1, dtype, 2.0)
    if len(set(new)) == 1:
        q = q.view(len(new), new[0], hq, d)
        got = pool.attend(q, lens, causal=causal, return_softmax_lse=True)
    else:
        cu = torch.tensor(starts_of(new), dtype=torch.int32).cuda()
        got = pool.attend(q, lens, causal=causal, return_softmax_lse=True, cu_seqlens_q=cu, max_seqlen_q=max(new))
    check_attend(pool, q, lens, new, got, causal)


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_attend_empty_and_short_caches(cache, n):
    """No rows, one row, fewer rows than tokens (the first tokens see nothing), lengths out of range."""
    lens = [0, 1, n - 1, n, 2 * n, -7, 2 ** 31 - 1]
    pool = Pool(len(lens), 6, 16, 2, 64, cache, seed=8)
    q = randn((len(lens), n, 4, 64), 1)
    got = pool.attend(q, lens, return_softmax_lse=True)
    check_attend(pool, q, [min(x, 96) for x in lens], [n] * len(lens), got)


def test_attend_no_pages():
    from flash_attn_legacy import flash_attn_with_paged_kvcache
    q = randn((2, 1, 4, 64), 1)
    cache = torch.empty((0, 16, 2, 64), dtype=torch.float16, device="cuda")
    table = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    o, lse = flash_attn_with_paged_kvcache(q, cache, cache, table, 0, return_softmax_lse=True)
    assert bool((o == 0).all()) and bool(torch.isneginf(lse).all())
    o = flash_attn_with_paged_kvcache(q[:0], cache, cache, table[:0], 0)
    assert o.shape == (0, 1, 4, 64)
    o = flash_attn_with_paged_kvcache(q[:, :0], cache, cache, table, 0)
    assert o.shape == (2, 0, 4, 64)


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("n", [1, 50])
def test_attend_stale_rows_and_missing_pages(cache, n):
    """Rows behind a sequence's last one and unused pages hold NaN; a page of the middle is missing."""
    lens = [75, 200]
    pool = Pool(2, 13, 16, 2, 128, cache, torch.bfloat16, seed=9)
    used = torch.zeros((pool.pages, 16), dtype=torch.bool)
    for b, m in enumerate(lens):
        for r in range(m):
            used[pool.table[b, r // 16], r % 16] = True
    for c in (pool.k_cache, pool.v_cache):
        (c.view(torch.uint8) if cache == "fp8" else c)[~used.cuda()] = 0x7f if cache == "fp8" else math.nan
    if cache == "fp8":
        for s in (pool.k_scale, pool.v_scale):
            s[~used.any(1).cuda()] = math.nan
    pool.table[1, 12:] = 2 ** 31 - 1           # entries past the length name anything
    q = randn((2, n, 8, 128), 1, torch.bfloat16)
    got = pool.attend(q, [75, 190], return_softmax_lse=True)
    check_attend(pool, q, [75, 190], [n, n], got)
    pool.table[0, 2], pool.table[1, 0] = -1, pool.pages
    got = pool.attend(q, lens[:1] + [190], return_softmax_lse=True)
    check_attend(pool, q, lens[:1] + [190], [n, n], got)


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("rows", [40, 3000])
@pytest.mark.parametrize("n", [1, 3, 12, 40])
def test_attend_not_finite(cache, rows, n):
    """A NaN key makes the tokens that see it NaN and no others; an infinite value is infinite in the
    result; the other sequence's rows are as they were."""
    pool = Pool(2, rows // 16 + 2, 16, 2, 64, cache, torch.bfloat16, seed=20)
    q = randn((2, n, 8, 64), 1, torch.bfloat16, 0.05)
    lens = [rows, rows - 3]
    clean = pool.attend(q, lens, return_softmax_lse=True)
    at, slot = int(pool.table[0, (rows - 1) // 16]), (rows - 1) % 16
    pool.rows(pool.k_cache)[at, slot, 0, 7] = math.nan            # the last row, KV head 0
    o, lse = pool.attend(q, lens, return_softmax_lse=True)
    assert bool(torch.isnan(o[0, -1, :4]).all()) and bool(torch.isnan(lse[0, -1, :4]).all())
    for a, b in ((o, clean[0]), (lse, clean[1])):
        assert torch.equal(a[1], b[1]) and torch.equal(a[0, :, 4:], b[0, :, 4:]) and torch.equal(a[0, :-1], b[0, :-1])
    pool.rows(pool.k_cache)[at, slot, 0, 7] = 0
    clean = pool.attend(q, lens, return_softmax_lse=True)
    # values: the last row, which the last token alone sees, and an early one
    near = 4 * 2.0 ** -8 * float(pool.rows(pool.v_cache).float().abs().max()) * (1 if cache == "same" else 2.0 ** -4)
    early = int(pool.table[1, 0])
    pool.rows(pool.v_cache)[at, slot, 0, 5] = math.nan
    if cache == "same":
        pool.rows(pool.v_cache)[early, 2, 1, 5] = math.inf
    o, lse = pool.attend(q, lens, return_softmax_lse=True)
    want_nan, want_inf = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(o, dtype=torch.bool)
    want_nan[0, -1, :4, 5] = True
    for i in range(n):
        want_inf[1, i, 4:, 5] = cache == "same" and lens[1] - n + i >= 2
    assert torch.equal(torch.isnan(o), want_nan) and torch.equal(o == math.inf, want_inf)
    rest = ~(want_nan | want_inf)
    # two results of rounded probabilities: each within 2 u of sum p |v| <= max |v|
    assert float((o.float() - clean[0].float()).abs()[rest].max()) <= near
    seen = torch.isfinite(clean[1])
    assert torch.equal(torch.isfinite(lse), seen) and float((lse - clean[1])[seen].abs().max()) <= 1e-4


@pytest.mark.parametrize("n", [1, 5])
def test_attend_hundreds_of_sequences(n):
    """More sequences than are read at once, some of them empty, in runs that hold many of them."""
    g = torch.Generator().manual_seed(5)
    lens = [int(x) if int(x) > 20 else 0 for x in torch.randint(0, 130, (700,), generator=g)]
    lens[3], lens[699] = 2100, 2090
    pool = Pool(1, 2200, 16, 2, 32, "fp8", seed=21)
    table = torch.zeros((700, 132), dtype=torch.int32)
    at = 0
    for b, m in enumerate(lens):
        used = -(-m // 16)
        table[b, :used] = pool.table[0, at:at + used].cpu()
        at = (at + used) % 2000
    pool.table = table.cuda()
    q = randn((700, n, 4, 32), 1)
    check_attend(pool, q, lens, [n] * 700, pool.attend(q, lens, return_softmax_lse=True))


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("n", [1, 24])
def test_attend_many_sequences(cache, n):
    """More sequences than a wave has lanes, most of them short."""
    g = torch.Generator().manual_seed(3)
    lens = [int(x) for x in torch.randint(n, 90, (150,), generator=g)]
    lens[77] = 900
    pool = Pool(150, 29, 32, 1, 64, cache, seed=10)
    q = randn((150, n, 4, 64), 1)
    got = pool.attend(q, lens, return_softmax_lse=True)
    check_attend(pool, q, lens, [n] * 150, got)


@pytest.mark.parametrize("cache", ["fp8", "same"])
def test_attend_packed_rows_outside_every_sequence(cache):
    pool = Pool(3, 5, 16, 2, 64, cache, seed=11)
    q = randn((60, 4, 64), 1)
    # (the longest sequence's length only sizes the grid: 20 is the tile kernel, one column tile of two)
    for first, hint in ((4, 33), (0, 1), (0, 0), (4, 20), (4, 10 ** 9)):
        cu = torch.tensor([first, 9, 9, 42], dtype=torch.int32).cuda()
        lens = [30, 8, 77]
        o, lse = pool.attend(q, lens, cu_seqlens_q=cu, max_seqlen_q=hint, return_softmax_lse=True)
        check_attend(pool, q[first:42], lens, [9 - first, 0, 33], (o[first:42], lse[first:42]))
        for t in (slice(0, first), slice(42, 60)):
            assert bool((o[t] == 0).all()) and bool(torch.isneginf(lse[t]).all())


@pytest.mark.parametrize("n", [1, 40])
def test_attend_scales_far_apart(n):
    """Value scales that differ by 2^40 from page to page, a zero scale, a scale that is no power of
    two, and scores that are large and negative."""
    pool = Pool(2, 8, 16, 2, 64, "fp8", torch.bfloat16, seed=12)
    order = pool.table.long()
    pool.v_scale[order[0]] = torch.exp2(torch.tensor([-20., 20, 0, -20, 5, 20, -20, 1])).cuda()[:, None]
    pool.v_scale[order[1]] = torch.tensor([0.3, 1e-5, 3.0, 0.7, 1e-3, 0.11, 0.2, 5e3]).cuda()[:, None]
    pool.k_scale[order[1]] *= 1.7
    q = randn((2, n, 4, 64), 1, torch.bfloat16, 8.0)
    lens = [128, 115]
    check_attend(pool, q, lens, [n, n], pool.attend(q, lens, return_softmax_lse=True))
    check_attend(pool, q, lens, [n, n], pool.attend(q, lens, return_softmax_lse=True, softmax_scale=-0.2), scale=-0.2)
    pool.v_scale.zero_()
    o, lse = pool.attend(q, lens, return_softmax_lse=True)
    assert bool((o == 0).all()) and bool(torch.isfinite(lse).all())


def test_attend_three_dims_and_integer_lengths():
    pool = Pool(3, 4, 16, 2, 64, "fp8", seed=13)
    q = randn((3, 4, 64), 1)
    o, lse = pool.attend(q, 50, return_softmax_lse=True)
    assert o.shape == (3, 4, 64) and lse.shape == (3, 4)
    check_attend(pool, q, [50] * 3, [1] * 3, (o, lse))
    long = torch.tensor([50, 50, 50])
    assert torch.equal(pool.attend(q, long), o)         # int64 on the host, as flash_attn_with_kvcache takes


def test_pools_past_32_bits():
    """Pages whose bytes lie past 2^32: written and read there."""
    from flash_attn_legacy import flash_attn_with_paged_kvcache, paged_kvcache_append
    pages, page, hkv, d = 70000, 64, 8, 128                    # 4.6 GB each
    k_cache, v_cache = (torch.zeros((pages, page, hkv, d), dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    scale = torch.ones((2, pages, hkv), device="cuda")
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32).cuda()
    for n in (1, 150):
        k, v = randn((1, n, hkv, d), n), randn((1, n, hkv, d), n + 1)
        q = randn((1, n, 16, d), n + 2)
        paged_kvcache_append(k, v, k_cache, v_cache, table, 10, scale[0], scale[1])
        got = flash_attn_with_paged_kvcache(q, k_cache, v_cache, table, 10 + n, scale[0], scale[1], return_softmax_lse=True)
        small = Pool(1, 3, page, hkv, d, "fp8")
        small.table = torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda()
        at = table[0].long()
        small.k_cache, small.v_cache, small.k_scale, small.v_scale = k_cache[at], v_cache[at], scale[0][at], scale[1][at]
        check_attend(small, q, [10 + n], [n], got)
        row = k_cache[pages - 1, 10].double() * scale[0, pages - 1][:, None]
        assert bool(((row - k[0, 0].double()).abs() <= torch.maximum(k[0, 0].double().abs() * 2.0 ** -4,
                                                                     scale[0, pages - 1][:, None].double() * 2.0 ** -10)).all())


# ---- both together ---------------------------------------------------------------------------

@pytest.mark.parametrize("cache", ["fp8", "same"])
def test_serving_loop(cache):
    """Prompts of odd lengths, a chunk behind them, proposed tokens of which some are taken back, and
    decode steps: each step's output follows from the rows that the cache holds, and those are the
    rotated keys and the values to the cache's precision."""
    from flash_attn_legacy import rotary_cos_sin
    dtype, d, hkv, hq, page = torch.bfloat16, 64, 2, 8, 16
    pool = Pool(3, 20, page, hkv, d, cache, dtype, seed=14)
    cos, sin = rotary_cos_sin(20 * page, d, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    kept = [[], [], []]
    steps = [[37, 1, 90], [20, 64, 5], [4, 4, 4], [1, 1, 1], [1, 1, 1], [1, 1, 1]]
    for s, new in enumerate(steps):
        total = sum(new)
        k, v, q = (randn((total, h, d), 10 * s + i, dtype) for i, h in enumerate((hkv, hkv, hq)))
        cu = torch.tensor(starts_of(new), dtype=torch.int32).cuda()
        shape = (lambda x: x) if s < 2 else (lambda x: x.view(3, new[0], *x.shape[1:]))
        kw, kwa = ({}, {}) if s >= 2 else (dict(cu_seqlens=cu, max_seqlen=max(new)), dict(cu_seqlens_q=cu, max_seqlen_q=max(new)))
        rq = pool.append(shape(k), shape(v), lens, q=shape(q), rotary_cos=cos, rotary_sin=sin, **kw)
        after = lens + (cu[1:] - cu[:-1])
        got = pool.attend(rq, after, return_softmax_lse=True, **kwa)
        check_attend(pool, rq, after.tolist(), new, got)
        for b, t0 in enumerate(starts_of(new)[:-1]):
            for i in range(new[b]):
                kept[b].append((orc.rotate(k[t0 + i].double(), int(lens[b]) + i, cos, sin, d, False), v[t0 + i].double()))
        if s == 2:                    # one proposed token of four is accepted
            after = lens + 1
            for rows in kept:
                del rows[-3:]
        lens = after
    for b in range(3):
        for r, (k, v) in enumerate(kept[b]):
            at, slot = int(pool.table[b, r // page]), r % page
            for c, sc, y in ((pool.k_cache, pool.k_scale, k), (pool.v_cache, pool.v_scale, v)):
                x = c[at, slot].double()
                if cache == "fp8":    # one rounding per growth of the page's scale, each half a step at most
                    x = x * sc[at].double()[:, None]
                    bound = torch.maximum(y.abs() * 2.0 ** -4, 2 * sc[at].double()[:, None] * 2.0 ** -10) + 1e-5
                else:
                    bound = y.abs() * 2.0 ** -8 + 1e-5
                assert bool(((x - y).abs() <= bound).all()), (b, r)


def test_prefill_equals_flash_attention():
    """A whole prompt through 16-bit pages gives what the packed kernel gives on the same rows."""
    from flash_attn_legacy import flash_attn_varlen_func
    new = [100, 257, 31]
    pool = Pool(3, 5, 64, 2, 128, "same", seed=15)
    k, v, q = randn((388, 2, 128), 1), randn((388, 2, 128), 2), randn((388, 8, 128), 3)
    cu = torch.tensor(starts_of(new), dtype=torch.int32).cuda()
    rq = pool.append(k, v, 0, q=q, cu_seqlens=cu, max_seqlen=257)
    o = pool.attend(rq, new, cu_seqlens_q=cu, max_seqlen_q=257)
    ref = flash_attn_varlen_func(q, k, v, cu, cu, 257, 257, causal=True)
    # two results of fp16 probabilities: each within 2 u of sum p |v| <= max |v|
    assert float((o.float() - ref.float()).abs().max()) <= 4 * 2.0 ** -11 * float(v.abs().max())


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("n", [1, 40])
def test_captured_steps(cache, n):
    """A step captured once and replayed while lengths and inputs change in place; two graphs at
    once; every replay equals the eager call."""
    from flash_attn_legacy import rotary_cos_sin
    pool, eager = (Pool(2, 30, 16, 2, 64, cache, seed=16) for _ in range(2))
    cos, sin = rotary_cos_sin(480, 64, device="cuda")
    lens = torch.tensor([11, 150], dtype=torch.int32).cuda()
    k, v, q = randn((2, n, 2, 64), 1), randn((2, n, 2, 64), 2), randn((2, n, 4, 64), 3)

    def step(p):
        rq = p.append(k, v, lens, q=q, rotary_cos=cos, rotary_sin=sin)
        return p.attend(rq, lens + n, return_softmax_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(Pool(2, 30, 16, 2, 64, cache, seed=16))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(pool))
        graphs.append(g)
    for r in range(4):
        k.copy_(randn(k.shape, 20 + r)), v.copy_(randn(v.shape, 30 + r)), q.copy_(randn(q.shape, 40 + r))
        junk = torch.randn(1 << 20, device="cuda").sum()
        torch.cuda.synchronize()
        graphs[r % 2].replay()
        want = step(eager)
        torch.cuda.synchronize()
        for a, b in zip(outs[r % 2], want):
            assert torch.equal(a, b)
        assert same(pool.k_cache, eager.k_cache) and same(pool.v_cache, eager.v_cache)
        lens += n
        del junk


def test_other_streams_and_repeats():
    """Calls on two streams at once, and the same call again, give the same bits."""
    pool = Pool(4, 60, 16, 2, 128, "fp8", torch.bfloat16, seed=17)
    q = randn((4, 1, 8, 128), 1, torch.bfloat16)
    lens = torch.tensor([900, 30, 500, 1], dtype=torch.int32).cuda()
    want = pool.attend(q, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(pool.attend(q, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---- ways of use -----------------------------------------------------------------------------

@pytest.mark.parametrize("cache", ["fp8", "same"])
def test_prompt_and_single_tokens_in_one_batch(cache):
    """A scheduler's step: one prompt's chunk packed with the tokens of running sequences and an
    empty one; the append and the attention behind it."""
    lens, new = [100, 37, 500, 0, 64, 15, 333, 1, 250], [1, 1, 300, 0, 1, 1, 1, 1, 1]
    pool = Pool(len(lens), 26, 32, 2, 128, cache, torch.bfloat16, seed=31)
    total, cu = sum(new), torch.tensor(starts_of(new), dtype=torch.int32).cuda()
    k, v, q = (randn((total, h, 128), i, torch.bfloat16) for i, h in enumerate((2, 2, 8)))
    before = snapshot(pool)
    assert torch.equal(pool.append(k, v, lens, q=q, cu_seqlens=cu, max_seqlen=300), q)
    check_append(pool, k, v, lens, new, before)
    after = [a + n for a, n in zip(lens, new)]
    got = pool.attend(q, after, return_softmax_lse=True, cu_seqlens_q=cu, max_seqlen_q=300)
    check_attend(pool, q, after, new, got)


FEW_AND_MANY = [
    # d, hkv, hq, dtype, lens (with the new rows), new
    (128, 2, 8, torch.bfloat16, [700, 5, 333, 90, 40, 3], [4, 5, 200, 1, 0, 3]),
    (256, 1, 2, torch.float16, [30, 150, 300, 1, 64, 77], [8, 9, 150, 1, 2, 1]),
    (64, 4, 4, torch.float16, [16, 290, 90, 33, 0], [16, 17, 90, 2, 1]),
    (96, 1, 20, torch.bfloat16, [1, 20, 100, 260, 65, 7], [1, 0, 30, 1, 2, 0]),
    (128, 2, 8, torch.float16, [600, 500, 40, 30, 5], [1, 12, 2, 0, 5]),
    (32, 8, 32, torch.float16, [100, 2100, 900], [1, 2048, 2]),
]


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", FEW_AND_MANY, ids=lambda c: f"d{c[0]}h{c[1]}-{c[2]}n{max(c[5])}")
def test_attend_few_and_many_tokens_packed(case, causal, cache):
    """Sequences around the number of tokens up to which another kernel takes them, rows outside
    every sequence, and the longest stated exactly, too long and too short."""
    d, hkv, hq, dtype, lens, new = case
    pool = Pool(len(lens), -(-max(lens) // 16) + 1, 16, hkv, d, cache, dtype, seed=d + hq)
    front, back = 3, 5
    cu = (torch.tensor(starts_of(new), dtype=torch.int32) + front).cuda()
    q = randn((front + sum(new) + back, hq, d), 1, dtype, 2.0)
    for longest in (max(new), q.shape[0], 2, max(new) // 2):
        o, lse = pool.attend(q, lens, causal=causal, return_softmax_lse=True, cu_seqlens_q=cu, max_seqlen_q=longest)
        for x in (slice(0, front), slice(-back, None)):
            assert bool((o[x] == 0).all()) and bool(torch.isneginf(lse[x]).all())
        check_attend(pool, q[front:-back], lens, new, (o[front:-back], lse[front:-back]), causal)


@pytest.mark.parametrize("cache", ["fp8", "same"])
@pytest.mark.parametrize("most", [1, 24])
def test_hundreds_of_packed_sequences(most, cache):
    """More sequences than are searched at once, of one token or of up to 24, long ones among them."""
    g = torch.Generator().manual_seed(most)
    n = 600
    new = torch.randint(0, most + 1, (n,), generator=g).tolist()
    new[0], new[299], new[599] = 70, 33, 90
    lens = torch.randint(0, 30, (n,), generator=g).tolist()
    pool = Pool(n, 8, 16, 1, 32, cache, seed=23)
    k, v, q = (randn((sum(new), h, 32), i) for i, h in enumerate((1, 1, 2)))
    starts = starts_of(new)
    tensor = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    before = snapshot(pool)
    pool.append(k, v, lens, cu_seqlens=tensor(starts), max_seqlen=max(new))
    got = snapshot(pool)
    for name, t in before.items():
        getattr(pool, name).copy_(t)
    table = pool.table
    for a in range(0, n, 200):   # the same in three calls
        t0, t1 = starts[a], starts[a + 200]
        pool.table = table[a:a + 200]
        pool.append(k[t0:t1], v[t0:t1], lens[a:a + 200], cu_seqlens=tensor([t - t0 for t in starts[a:a + 201]]), max_seqlen=90)
    pool.table = table
    for name, t in got.items():
        assert same(getattr(pool, name), t), name
    after = [x + y for x, y in zip(lens, new)]
    res = pool.attend(q, after, return_softmax_lse=True, cu_seqlens_q=tensor(starts), max_seqlen_q=max(new))
    check_attend(pool, q, after, new, res)


@pytest.mark.parametrize("cache", ["fp8", "same"])
def test_rejected_tokens_are_written_over(cache):
    """Speculative decoding: five tokens proposed, two kept, the next five start behind those."""
    pool = Pool(2, 3, 32, 2, 64, cache, seed=17)
    for step, lens in enumerate(([20, 30], [22, 32], [24, 33])):
        k, v = randn((10, 2, 64), 2 * step, scale=3.0 ** step), randn((10, 2, 64), 2 * step + 1, scale=9.0 - 4 * step)
        before = snapshot(pool)
        pool.append(k.view(2, 5, 2, 64), v.view(2, 5, 2, 64), lens)
        check_append(pool, k, v, lens, [5, 5], before)
        q = randn((2, 5, 4, 64), 50 + step)
        after = [n + 5 for n in lens]
        check_attend(pool, q, after, [5, 5], pool.attend(q, after, return_softmax_lse=True))


@pytest.mark.parametrize("n", [1, 9, 40])
def test_attend_shared_pages(n):
    """Sequences with one prefix read the same pages, keys and values may be one cache, and one
    page may stand in a table twice."""
    pool = Pool(3, 6, 32, 1, 64, "fp8", seed=5)
    pool.table[1:, :4] = pool.table[0, :4]
    pool.table[2, 4] = pool.table[2, 1]
    pool.v_cache, pool.v_scale = pool.k_cache, pool.k_scale
    q = randn((3, n, 4, 64), 3)
    lens = [190, 128 + n, 150]
    check_attend(pool, q, lens, [n] * 3, pool.attend(q, lens, return_softmax_lse=True))


# ---- refusals --------------------------------------------------------------------------------

def test_refusals():
    from flash_attn_legacy import flash_attn_with_paged_kvcache as attend, paged_kvcache_append as append
    pool = Pool(2, 2, 16, 2, 64, "fp8")
    kc, vc, ks, vs, table = pool.k_cache, pool.v_cache, pool.k_scale, pool.v_scale, pool.table
    k, q = randn((2, 1, 2, 64), 1), randn((2, 1, 4, 64), 2)
    before = snapshot(pool)

    def refused(match, fn, *a, **kw):
        with pytest.raises((RuntimeError, AssertionError), match=match):
            fn(*a, **kw)

    for fn, x in ((lambda *a, **kw: append(k, k, *a, **kw), k), (lambda *a, **kw: attend(q, *a, **kw), q)):
        refused("k_scale and v_scale", fn, kc, vc, table, 1)
        refused("k_scale and v_scale must be float32", fn, kc, vc, table, 1, ks[:1], vs)
        refused("k_scale and v_scale must be float32", fn, kc, vc, table, 1, ks.double(), vs)
        refused("for float8 caches", fn, kc.half(), vc.half(), table, 1, ks, vs)
        refused("must both be", fn, kc.bfloat16(), vc.bfloat16(), table, 1)
        refused("must both be", fn, kc, vc.half(), table, 1, ks, vs)
        refused("shape mismatch", fn, kc, vc[:-1], table, 1, ks, vs)
        refused("page_table must be", fn, kc, vc, table[:1], 1, ks, vs)
        refused("page_table must be", fn, kc, vc, table[0], torch.ones(2, dtype=torch.int32), ks, vs)
        refused("must hold 2 lengths", fn, kc, vc, table, torch.ones(3, dtype=torch.int32).cuda(), ks, vs)
        refused("page_size must be a multiple of 16", fn, kc[:, :8], vc[:, :8], table, 1, ks, vs)
        refused("contiguous in the head", fn, kc.transpose(2, 3).contiguous().transpose(2, 3),
                vc.transpose(2, 3).contiguous().transpose(2, 3), table, 1, ks, vs)
        refused("multiple of 16 bytes", fn, torch.empty((7, 16, 2, 72), dtype=torch.uint8, device="cuda").view(FP8)[..., :64],
                torch.empty((7, 16, 2, 72), dtype=torch.uint8, device="cuda").view(FP8)[..., :64], table, 1, ks, vs)
        refused("must be on cuda", fn, kc.cpu(), vc, table, 1, ks, vs)
        refused("unknown cache_layout", fn, kc, vc, table, 1, ks, vs, cache_layout="hsbd")
    refused("go together", append, k, k, kc, vc, table, 1, ks, vs, max_seqlen=1)
    refused("float16 or bfloat16", append, k.float(), k.float(), kc, vc, table, 1, ks, vs)
    refused("head_dim must be", append, k[..., :48], k[..., :48], kc, vc, table, 1, ks, vs)
    refused("v must have", append, k, k[:, :, :1], kc, vc, table, 1, ks, vs)
    refused("different numbers of heads", append, q, q, kc, vc, table, 1, ks, vs)
    refused("q must have", append, k, k, kc, vc, table, 1, ks, vs, q=q[:1])
    refused("divisible", append, k, k, kc, vc, table, 1, ks, vs, q=randn((2, 1, 3, 64), 1))
    cos = torch.ones((32, 32), device="cuda")
    refused("go together", append, k, k, kc, vc, table, 1, ks, vs, rotary_cos=cos)
    refused("31 rows for the 32 positions", append, k, k, kc, vc, table, 1, ks, vs, rotary_cos=cos[:31], rotary_sin=cos[:31])
    refused("float32", append, k, k, kc, vc, table, 1, ks, vs, rotary_cos=cos.half(), rotary_sin=cos.half())
    refused("multiple of 16", append, k, k, kc, vc, table, 1, ks, vs, rotary_cos=cos[:, :4], rotary_sin=cos[:, :4])
    wide = torch.ones((32, 40), device="cuda")
    refused("up to head_dim", append, k, k, kc, vc, table, 1, ks, vs, rotary_cos=wide, rotary_sin=wide)
    refused("must not share", append, k, k, kc, kc, table, 1, ks, vs)
    refused("must not share", append, k, k, kc, vc, table, 1, ks, ks)
    refused("rows overlap", append, k, k, kc[:1].expand(7, -1, -1, -1), vc, table, 1, ks, vs)
    refused("entries overlap", append, k, k, kc, vc, table, 1, ks[:1].expand(7, -1), vs)
    refused("divisible", attend, randn((2, 1, 3, 64), 1), kc, vc, table, 1, ks, vs)
    refused(r"q must be \[total", attend, q, kc, vc, table, 1, ks, vs, cu_seqlens_q=torch.zeros(3, dtype=torch.int32).cuda(),
            max_seqlen_q=1)
    refused("tokens without a sequence", attend, q[:, 0], kc, vc, table[:0], 1, ks, vs,
            cu_seqlens_q=torch.zeros(1, dtype=torch.int32).cuda(), max_seqlen_q=1)
    torch.cuda.synchronize()
    for name, t in before.items():
        assert same(getattr(pool, name), t), name
