"""The paged-cache operators whose speed this repository is measured by.

Two operators: `paged_kvcache_append` (rotate keys and queries, write keys and values into a
paged cache in 16 or 8 bits) and `flash_attn_with_paged_kvcache` (attention of one or more new
tokens per sequence to that cache).  A case is one call, or one decode step's pair of calls.
`listed()` holds fixed cases, `draw(rng)` samples the ranges they stand for.  The file is
imported with the repository's root as the working folder.
"""

import math
import os
import sys

import torch

own = False   # True: the framework's kernels; False: the same in elementary torch operations

# Upper ends of what a drawn case may cost; both lie below the largest listed cases.
_MAX_FLOPS = 3.0e11
_MAX_BYTES = 1.0e9
_MAX_SCORES = 1.2e9      # elements of the plain form's score matrix

_E4M3_MAX = 448.0        # largest finite value of float8_e4m3fn
_MIN_EXP = -126          # smallest exponent of a page's scale


def listed():
    return [
        # One user's chat step: one token is rotated and appended to an 8-bit cache of 1000 rows.
        # Launch and latency.
        dict(name="append8_token", kind="append", batch=1, min_new=1, max_new=1, min_len=1000, max_len=1000,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="bfloat16", layout="bshd", rotary=128,
             interleaved=False, packed=False),
        # A serving step of 32 users (the benchmark's decode configuration): every sequence gets
        # one token, somewhere inside a page.
        dict(name="append8_batch", kind="append", batch=32, min_new=1, max_new=1, min_len=1024, max_len=32768,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="float16", layout="bshd", rotary=128,
             interleaved=False, packed=False),
        # 16 packed prompts of 64 to 4096 tokens (the benchmark's packed batch) into an empty 8-bit cache.
        dict(name="append8_prompts", kind="append", batch=16, min_new=64, max_new=4096, min_len=0, max_len=0,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="bfloat16", layout="bshd", rotary=128,
             interleaved=False, packed=True),
        # Chunks of odd lengths behind odd prefixes, 16-bit cache of small pages in the head-major
        # layout, half of each head rotated, in interleaved pairs.
        dict(name="append16_chunks", kind="append", batch=6, min_new=37, max_new=1531, min_len=11, max_len=2000,
             heads_q=16, heads_kv=16, dim=64, page=16, cache="same", dtype="float16", layout="bhsd", rotary=32,
             interleaved=True, packed=True),
        # One user's chat step against 1000 rows held in 8 bits: launches and latency.
        dict(name="decode8_token", kind="attend", batch=1, min_new=1, max_new=1, min_len=1000, max_len=1000,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="bfloat16", layout="bshd", causal=True,
             packed=False),
        # The benchmark's decode configuration on an 8-bit paged cache: bound by reading it.
        dict(name="decode8_batch", kind="attend", batch=32, min_new=1, max_new=1, min_len=1024, max_len=32768,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="float16", layout="bshd", causal=True,
             packed=False),
        # 24 users of a model with 64-wide heads and one KV head each, 16-bit cache of small pages.
        dict(name="decode16_mha", kind="attend", batch=24, min_new=1, max_new=1, min_len=77, max_len=4099,
             heads_q=12, heads_kv=12, dim=64, page=16, cache="same", dtype="float16", layout="bhsd", causal=True,
             packed=False),
        # A decode step as a serving loop runs it, append then attention, one layer of 16 users.
        dict(name="step8", kind="step", batch=16, min_new=1, max_new=1, min_len=500, max_len=8000,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="bfloat16", layout="bshd", rotary=128,
             interleaved=False, causal=True, packed=False),
        # Speculative decoding: five proposed tokens of 8 users are checked in one pass.
        dict(name="verify8", kind="attend", batch=8, min_new=5, max_new=5, min_len=700, max_len=6000,
             heads_q=32, heads_kv=8, dim=128, page=32, cache="fp8", dtype="bfloat16", layout="bshd", causal=True,
             packed=False),
        # A 1024-token chunk of a long prompt behind 8192 cached rows (chunked prefill).
        dict(name="chunk8", kind="attend", batch=1, min_new=1024, max_new=1024, min_len=9216, max_len=9216,
             heads_q=32, heads_kv=8, dim=128, page=64, cache="fp8", dtype="bfloat16", layout="bshd", causal=True,
             packed=True),
        # A packed mixed batch: short and long chunks of odd lengths on 16-bit pages, 96-wide heads.
        dict(name="chunks16", kind="attend", batch=5, min_new=3, max_new=1201, min_len=1300, max_len=3001,
             heads_q=16, heads_kv=4, dim=96, page=32, cache="same", dtype="float16", layout="bhsd", causal=True,
             packed=True),
        # The last tokens of long prompts on the widest heads.
        dict(name="chunk8_d256", kind="attend", batch=2, min_new=511, max_new=511, min_len=4000, max_len=6001,
             heads_q=16, heads_kv=8, dim=256, page=128, cache="fp8", dtype="float16", layout="bshd", causal=True,
             packed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above: each kind, all head dims with 64 and 128 most often,
    both cache types and element types, lengths over three orders of magnitude."""
    while True:
        kind = rng.choice(["append", "append", "attend", "attend", "attend", "step"])
        heads_q, heads_kv = rng.choice([(8, 8), (16, 16), (12, 12), (32, 8), (32, 8), (32, 8), (16, 8), (16, 4), (8, 1),
                                        (28, 4), (40, 8)])
        dim = rng.choice([32, 64, 64, 64, 96, 128, 128, 128, 128, 256])
        case = dict(kind=kind, batch=_log_int(rng, 1, 80), heads_q=heads_q, heads_kv=heads_kv, dim=dim,
                    page=rng.choice([16, 32, 64, 64, 128, 256]), cache=rng.choice(["fp8", "fp8", "same"]),
                    dtype=rng.choice(["float16", "bfloat16"]), layout=rng.choice(["bshd", "bhsd"]))
        many = kind != "step" and rng.random() < 0.5
        hi = _log_int(rng, 2, 2048) if many else rng.choice([1, 1, 1, 2, 4, 7])
        case.update(max_new=hi, min_new=rng.choice([hi, max(1, hi // 7)]), packed=many and rng.random() < 0.7)
        if not case["packed"]:
            case["min_new"] = hi
        top = _log_int(rng, 16, 32768)
        low = rng.choice([top, top // 8])
        if kind == "append":
            low, top = (0, 0) if many and rng.random() < 0.5 else (low, top)
        else:       # the cache already holds the new rows
            low, top = low + hi, top + hi
        case.update(min_len=low, max_len=top)
        if kind != "append":
            case["causal"] = kind == "step" or rng.random() < 0.8
        if kind != "attend":
            case.update(rotary=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3)
        if case.get("rotary", 16) % 16:
            continue
        scores = case["batch"] * heads_q * float(hi) * (top + case["page"])
        w = work(case)
        if (w["flops"] < _MAX_FLOPS and 2.0e4 < w["bytes"] < _MAX_BYTES and (kind == "append" or scores < _MAX_SCORES)
                and case["batch"] * float(top + hi) * heads_kv * dim < _MAX_BYTES):
            return case


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi] in a scrambled order, the ends included."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 11, 13, 17, 19, 23) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * (i * step % n) // (n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, cache rows given to the call) of every sequence.  An append's rows are those
    before it; attention's rows include the new tokens; a step's are those before it."""
    n = case["batch"]
    new = _spread(case["min_new"], case["max_new"], n)
    rows = _spread(case["min_len"], case["max_len"], n)
    return new, rows


def _total_rows(case):
    new, rows = _lengths(case)
    return [r + (n if case["kind"] != "attend" else 0) for n, r in zip(new, rows)]


def work(case):
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    cb = 1 if case["cache"] == "fp8" else 2
    new, rows = _lengths(case)
    t = float(sum(new))
    bytes_ = flops = 0.0
    if case["kind"] != "attend":
        # q, k, v and the rotation's rows in; rotated q and the cache rows out
        bytes_ += 2 * t * d * (hq + 2 * hkv) + 4 * t * case["rotary"] + 2 * t * d * hq + 2 * t * d * hkv * cb
        flops += 3 * t * case["rotary"] * (hq + hkv) + (2 * t * d * hkv if cb == 1 else 0)
    if case["kind"] != "append":
        total = _total_rows(case)
        # the cache's rows, q in and o out
        bytes_ += 2.0 * hkv * d * cb * sum(total) + 4 * t * d * hq
        pairs = sum(float(n) * m - (n * (n - 1) / 2 if case["causal"] else 0) for n, m in zip(new, total))
        flops += 4 * hq * d * pairs
    return dict(bytes=bytes_, flops=flops)


def _page_scale(amax):
    """The power of two that a page of this largest magnitude is stored in units of: the
    smallest one, from 2^-126 on, in which 448 units reach it."""
    m, x = torch.frexp(amax)
    e = torch.where(amax > 0, x - 9 + (m > 0.875).to(x.dtype), torch.full_like(x, _MIN_EXP)).clamp(min=_MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _quantise(x, scale):
    return (x * (1 / scale)).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def _inputs(case, seed):
    """Activations as they reach attention: queries and values of about unit size, keys with a few
    large channels, heads of different magnitudes; pages in the order in which an allocator
    that has been running for a while hands them out."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    hq, hkv, d, p, b = case["heads_q"], case["heads_kv"], case["dim"], case["page"], case["batch"]
    new, rows = _lengths(case)
    total = _total_rows(case)
    per = [-(-m // p) for m in total]                      # pages of each sequence
    width = max(per)
    count = sum(per) + 1
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    first = torch.tensor([0] + per).cumsum(0)[:-1].cuda()
    col = torch.arange(width, device="cuda")
    held = col[None] < torch.tensor(per).cuda()[:, None]
    table = torch.where(held, order[(first[:, None] + col).clamp(max=count - 1)], order[-1])
    rnd = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    big = 1 + 3 * (torch.rand((hkv, d), generator=gen, device="cuda") < 0.03)
    size = torch.exp2(0.5 * rnd(2, hkv, 1))
    x = dict(table=table.contiguous(), lens=torch.tensor(rows, dtype=torch.int32).cuda())
    cache_type = torch.float8_e4m3fn if case["cache"] == "fp8" else dtype
    for name, factor in (("k", big * size[0]), ("v", size[1].expand(hkv, d))):
        full = torch.empty((count, p, hkv, d) if case["layout"] == "bshd" else (count, hkv, p, d), dtype=cache_type,
                           device="cuda")
        pages = full if case["layout"] == "bshd" else full.transpose(1, 2)
        scales = torch.empty((count, hkv), device="cuda")
        step = max(1, (1 << 27) // (p * hkv * d))
        for i in range(0, count, step):
            y = rnd(min(step, count - i), p, hkv, d) * factor
            if case["cache"] == "fp8":
                scales[i:i + step] = _page_scale(y.abs().amax((1, 3)))
                y = _quantise(y, scales[i:i + step, None, :, None])
            pages[i:i + step] = y.to(cache_type)
        x[name + "_cache"] = full
        x[name + "_scale"] = scales if case["cache"] == "fp8" else None
        if case["kind"] != "attend":
            y = (rnd(sum(new), hkv, d) * factor).to(dtype)
            x[name] = y if case["packed"] else y.view(b, new[0], hkv, d)
    q = rnd(sum(new), hq, d).to(dtype)
    x["q"] = q if case["packed"] else q.view(b, new[0], hq, d)
    x["cu"] = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda() if case["packed"] else None
    if case["kind"] != "attend":
        # angles of every position that the table's pages can hold, in 64 bits
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(width * p, dtype=torch.float64, device="cuda")[:, None] * freq
        x["cos"], x["sin"] = angle.cos().float(), angle.sin().float()
    return x


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    state["max_new"] = case["max_new"]
    if case["kind"] == "step":
        state["lens_after"] = state["lens"] + case["max_new"]
    if case["packed"]:      # the token's sequence and place, which a program that packs them has
        new = torch.tensor(_lengths(case)[0], device="cuda")
        state["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new)
        state["place"] = torch.arange(len(state["seq"]), device="cuda") - state["cu"][:-1].long()[state["seq"]]
    return state


# ---- plain forms -------------------------------------------------------------------------

def _rotate(x, cos, sin, case):
    """x [tokens, heads, d] in fp32, cos and sin [tokens, rotary / 2]"""
    r, half = case["rotary"], case["rotary"] // 2
    cos, sin = cos[:, None], sin[:, None]
    y = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :half], x[..., half:r]
        y[..., :half], y[..., half:r] = a * cos - b * sin, b * cos + a * sin
    return y


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _store8(cache, scale, y, page, slot, pages, fresh, before):
    """Rows y [tokens, heads, d] into (page, slot) of an 8-bit cache [pages, slots, heads, d].
    pages [m]: the pages they touch, fresh [m]: filled from their first slot on, before [m]:
    rows that were there."""
    amax = torch.zeros_like(scale)
    size = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y)).amax(-1)
    amax.scatter_reduce_(0, page[:, None].expand_as(size), size, "amax")
    need, old = _page_scale(amax[pages]), scale[pages]
    new = torch.where(fresh[:, None], need, torch.maximum(old, need))
    codes = cache[pages]
    again = _quantise(codes.float() * old[:, None, :, None], new[:, None, :, None])
    kept = (torch.arange(cache.shape[1], device=cache.device)[None] < before[:, None])[:, :, None, None]
    raised = (new > old)[:, None, :, None]
    _bytes(cache)[pages] = torch.where(kept & raised, _bytes(again), _bytes(codes))
    scale[pages] = new
    _bytes(cache)[page, slot] = _bytes(_quantise(y, scale[page][..., None]))


def _append_plain(s):
    case = s["case"]
    p, b = case["page"], case["batch"]
    seq_major = lambda t: t if case["layout"] == "bshd" else t.transpose(1, 2)
    flat = lambda t: t.float().reshape(-1, *t.shape[-2:])
    if case["packed"]:
        seq, place = s["seq"], s["place"]
        new = (s["cu"][1:] - s["cu"][:-1]).long()
    else:
        n = s["k"].shape[1]
        seq = torch.arange(b, device="cuda").repeat_interleave(n)
        place = torch.arange(n, device="cuda").repeat(b)
        new = torch.full((b,), n, device="cuda")
    lens = s["lens"].long()
    pos = lens[seq] + place
    page, slot = s["table"][seq, pos // p].long(), pos % p
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(flat(s["q"]), cos, sin, case).to(s["q"].dtype).view(s["q"].shape)
    k, v = _rotate(flat(s["k"]), cos, sin, case), flat(s["v"])
    kc, vc = seq_major(s["k_cache"]), seq_major(s["v_cache"])
    if case["cache"] != "fp8":
        kc[page, slot] = k.to(kc.dtype)
        vc[page, slot] = v.to(vc.dtype)
        return q, s["k_cache"], s["v_cache"]
    # the pages that the new rows touch; places past a sequence's last one name its first again
    most = (s["max_new"] + p - 2) // p + 1
    at = (lens // p)[:, None] + torch.arange(most, device="cuda")
    at = torch.where(at <= ((lens + new - 1) // p)[:, None], at, at[:, :1])
    pages = s["table"].gather(1, at).long().flatten()
    before = (lens[:, None] - at * p).clamp(min=0).flatten()
    for_k = (kc, s["k_scale"], k, page, slot, pages, before == 0, before)
    for_v = (vc, s["v_scale"], v, page, slot, pages, before == 0, before)
    _store8(*for_k)
    _store8(*for_v)
    return q, s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]


def _attend_plain(s, q, lens):
    case = s["case"]
    b, p, hq, hkv, d = case["batch"], case["page"], case["heads_q"], case["heads_kv"], case["dim"]
    width, n, dtype = s["table"].shape[1], s["max_new"], q.dtype
    table = s["table"].long()

    def rows(cache, scale):
        t = cache[table].float()                          # [B, pages, ...]
        t = t if case["layout"] == "bshd" else t.transpose(2, 3)
        if scale is not None:
            t = t * scale[table][:, :, None, :, None]
        return t.reshape(b, width * p, hkv, d).transpose(1, 2)

    if case["packed"]:
        new = s["cu"][1:] - s["cu"][:-1]
        full = torch.zeros((b, n, hq, d), device="cuda")
        full[s["seq"], s["place"]] = q.float()
    else:
        new = torch.full((b,), n, device="cuda", dtype=torch.int32)
        full = q.float()
    k, v = rows(s["k_cache"], s["k_scale"]), rows(s["v_cache"], s["v_scale"])
    full = full.view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    x = torch.matmul(full, k.transpose(2, 3)).mul_(1 / math.sqrt(d)).view(b, hkv, hq // hkv, n, width * p)
    end = lens[:, None].expand(b, n)
    if case["causal"]:
        end = end - new[:, None] + torch.arange(n, device="cuda")[None] + 1
    x.masked_fill_(torch.arange(width * p, device="cuda") >= end[:, None, None, :, None], -math.inf)
    most = x.amax(-1, keepdim=True).clamp(min=-3.0e38)
    x = x.sub_(most).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hkv, -1, width * p), v).view(b, hkv, hq // hkv, n, d) / total.clamp(min=1e-30)
    lse = (most + total.log())[..., 0].permute(0, 3, 1, 2).reshape(b, n, hq)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)
    if case["packed"]:
        return o[s["seq"], s["place"]].to(dtype), lse[s["seq"], s["place"]]
    return o.to(dtype), lse


# ---- the framework's calls ---------------------------------------------------------------

def _framework():
    root = os.path.join(os.getcwd(), "flash-attention-legacy_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import flash_attn_legacy
    return flash_attn_legacy


def _append_own(s):
    case, f = s["case"], _framework()
    q = f.paged_kvcache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                               k_scale=s["k_scale"], v_scale=s["v_scale"], q=s["q"], cu_seqlens=s["cu"],
                               max_seqlen=s["max_new"] if case["packed"] else None, rotary_cos=s["cos"],
                               rotary_sin=s["sin"], rotary_interleaved=case["interleaved"], cache_layout=case["layout"])
    if case["cache"] != "fp8":
        return q, s["k_cache"], s["v_cache"]
    return q, s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]


def _attend_own(s, q, lens):
    case, f = s["case"], _framework()
    return f.flash_attn_with_paged_kvcache(q, s["k_cache"], s["v_cache"], s["table"], lens, k_scale=s["k_scale"],
                                           v_scale=s["v_scale"], cu_seqlens_q=s["cu"],
                                           max_seqlen_q=s["max_new"] if case["packed"] else None, causal=case["causal"],
                                           return_softmax_lse=True, cache_layout=case["layout"])


def run(state):
    kind = state["case"]["kind"]
    append, attend = (_append_own, _attend_own) if own else (_append_plain, _attend_plain)
    if kind == "append":
        return append(state)
    if kind == "attend":
        return attend(state, state["q"], state["lens"])
    updated = append(state)
    return (*attend(state, updated[0], state["lens_after"]), *updated[1:])


# ---- the definition in 64 bits -----------------------------------------------------------

def _exact_append(case, x):
    """(rotated queries, K cache, K scales, V cache, V scales) after the append, row by page."""
    new, rows = _lengths(case)
    p, r, half = case["page"], case["rotary"], case["rotary"] // 2
    starts = torch.tensor([0] + new).cumsum(0).tolist()
    table = x["table"].cpu()
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    one = torch.arange(r, device="cuda")
    if case["interleaved"]:
        mate, pair, sign = one ^ 1, one // 2, torch.where(one % 2 == 0, -1.0, 1.0).double()
    else:
        mate, pair, sign = (one + half) % r, one % half, torch.where(one < half, -1.0, 1.0).double()

    def turned(t, at):
        t = t.double()
        angle = (torch.arange(at, at + t.shape[0], device="cuda").double()[:, None] * freq)[:, pair][:, None]
        y = t.clone()
        y[..., :r] = t[..., :r] * angle.cos() + sign * t[..., mate] * angle.sin()
        return y

    flat = {n: x[n].reshape(-1, *x[n].shape[-2:]) for n in ("q", "k", "v")}
    out = [torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")]
    turned_q = out[0].view(flat["q"].shape)
    caches = [(x[n + "_cache"].double(), None if x[n + "_scale"] is None else x[n + "_scale"].double()) for n in "kv"]
    for b in range(case["batch"]):
        lo, hi = starts[b], starts[b + 1]
        turned_q[lo:hi] = turned(flat["q"][lo:hi], rows[b])
        fresh = (turned(flat["k"][lo:hi], rows[b]), flat["v"][lo:hi].double())
        for y, (cache, scale) in zip(fresh, caches):
            at = 0
            while at < hi - lo:
                slot, page = (rows[b] + at) % p, int(table[b, (rows[b] + at) // p])
                n = min(p - slot, hi - lo - at)
                part = y[at:at + n].transpose(0, 1)                       # [heads, n, d]
                held = cache[page] if case["layout"] == "bhsd" else cache[page].transpose(0, 1)
                if scale is not None:
                    e = torch.ceil(torch.log2(part.abs().amax((1, 2)) / _E4M3_MAX)).clamp(min=_MIN_EXP)
                    unit = torch.exp2(e) if slot == 0 else torch.maximum(torch.exp2(e), scale[page])
                    held[:, :slot] *= (scale[page] / unit)[:, None, None]
                    scale[page] = unit
                    part = part / unit[:, None, None]
                held[:, slot:slot + n] = part
                at += n
    for cache, scale in caches:
        out += [cache] if scale is None else [cache, scale]
    return tuple(out)


def _exact_attend(case, x, q, caches, rows):
    new, _ = _lengths(case)
    p, group = case["page"], case["heads_q"] // case["heads_kv"]
    starts = torch.tensor([0] + new).cumsum(0).tolist()
    flat = q.double().reshape(-1, case["heads_q"], case["dim"])
    o = torch.empty(flat.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(flat.shape[:2], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        lo, hi, m = starts[b], starts[b + 1], rows[b]
        pages = x["table"][b, :-(-m // p)].long()
        seen = torch.full((hi - lo,), m, device="cuda")
        if case["causal"]:
            seen = m - (hi - lo) + 1 + torch.arange(hi - lo, device="cuda")
        hidden = torch.arange(m, device="cuda")[None] >= seen[:, None]
        for h in range(case["heads_kv"]):
            k, v = ((c[pages, :, h] if case["layout"] == "bshd" else c[pages, h]).double()
                    * (1.0 if s is None else s[pages, h].double()[:, None, None]) for c, s in caches)
            k, v = k.reshape(-1, case["dim"])[:m], v.reshape(-1, case["dim"])[:m]
            for g in range(h * group, (h + 1) * group):
                z = (flat[lo:hi, g] @ k.T / math.sqrt(case["dim"])).masked_fill_(hidden, -math.inf)
                lse[lo:hi, g] = torch.logsumexp(z, -1)
                o[lo:hi, g] = torch.softmax(z, -1) @ v
    return o.view(q.shape), lse.view(q.shape[:-1])


def exact(case, seed):
    """What `run` returns, in 64 bits.  A step's attention is taken over the cache that its append
    leaves, which holds rounded rows: that pair has no value of its own in 64 bits."""
    x = _inputs(case, seed)
    caches = [(x[n + "_cache"], x[n + "_scale"]) for n in "kv"]
    if case["kind"] == "attend":
        return _exact_attend(case, x, x["q"], caches, _lengths(case)[1])
    updated = _exact_append(case, x)
    return updated if case["kind"] == "append" else (None, None, *updated[1:])
