"""Paged KV cache on a CPU-only host: the C entry points' refusals, the Python layer's argument
checks, the rotation tables, and the 64-bit oracle against closed forms."""

import ctypes
import math

import pytest
import torch

FAL_OK, FAL_ERR_INVALID, FAL_ERR_UNSUPPORTED, FAL_ERR_LAUNCH, FAL_ERR_WORKSPACE = range(5)
P = 4096     # an aligned address that no call gets as far as using
V = P + (1 << 40)     # the values' cache and scales


def s3(*v):
    return (ctypes.c_int64 * 3)(*v)


def cache(ext, **kw):
    page, hkv, d = kw.get("page_size", 64), kw.get("heads_kv", 2), kw.get("head_dim", 128)
    c = ext.PagedCache(k=P, v=V, k_scale=P, v_scale=V, page_table=P, cache_seqlens=P, table_stride=4, batch=3,
                       seqlen=1, total_tokens=3, heads_q=8, heads_kv=2, head_dim=128, num_pages=10, page_size=64,
                       max_pages=4, fp8=1)
    c.k_strides[:] = c.v_strides[:] = (page * hkv * d, d, hkv * d)
    c.k_scale_strides[:] = c.v_scale_strides[:] = (hkv, 1)
    for name, value in kw.items():
        if name.endswith("strides"):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


@pytest.fixture(scope="module")
def ext():
    from flash_attn_legacy import hip_ext
    return hip_ext


def append(ext, c, k=P, q=P, q_out=P, strides=None, cos=P, rows=256, cos_stride=64, rotary=128, bf16=False):
    st = strides or s3(2048, 128, 1024)
    fn = ext._lib.fal_paged_append_bf16 if bf16 else ext._lib.fal_paged_append
    rc = fn(ctypes.byref(c) if c else None, k, P, q, q_out, st, st, st, st, cos, cos, rows, cos_stride, cos_stride,
            rotary, 0, None)
    return rc, ext._lib.fal_last_error().decode()


def attn(ext, c, q=P, o=P, strides=None, ws=0, bf16=False):
    st = strides or s3(2048, 128, 1024)
    fn = ext._lib.fal_paged_attn_bf16 if bf16 else ext._lib.fal_paged_attn
    rc = fn(ctypes.byref(c) if c else None, q, o, None, st, st, 0.1, 1, P if ws else None, ws, None)
    return rc, ext._lib.fal_last_error().decode()


BAD_CACHES = [
    (dict(head_dim=48), FAL_ERR_UNSUPPORTED, "head_dim must be 32, 64, 96, 128, or 256, got 48"),
    (dict(heads_q=7), FAL_ERR_INVALID, "divisible"),
    (dict(heads_kv=0), FAL_ERR_INVALID, "invalid sizes"),
    (dict(batch=-1), FAL_ERR_INVALID, "invalid sizes"),
    (dict(total_tokens=4), FAL_ERR_INVALID, "total_tokens must be batch * seqlen"),
    (dict(batch=0, seqlen=1, total_tokens=2, cu_seqlens=P), FAL_ERR_INVALID, "tokens without a sequence"),
    (dict(page_size=40), FAL_ERR_UNSUPPORTED, "page_size must be a multiple of 16"),
    (dict(page_size=0), FAL_ERR_UNSUPPORTED, "page_size must be a multiple of 16"),
    (dict(max_pages=2 ** 25), FAL_ERR_INVALID, "must not pass 2^30"),
    (dict(cache_seqlens=None), FAL_ERR_INVALID, "cache_seqlens: null pointer"),
    (dict(page_table=None), FAL_ERR_INVALID, "page_table: null pointer"),
    (dict(table_stride=-1), FAL_ERR_INVALID, "page_table: negative stride"),
    (dict(k=None), FAL_ERR_INVALID, "k_cache: null pointer"),
    (dict(v=P + 8), FAL_ERR_INVALID, "v_cache: base pointer must be 16-byte aligned"),
    (dict(k_strides=(16384, 128, 264)), FAL_ERR_INVALID, "k_cache: stride[2]=264 must be a non-negative multiple of 16 bytes"),
    (dict(v_strides=(-16384, 128, 256)), FAL_ERR_INVALID, "v_cache: stride[0]"),
    (dict(k_strides=(2 ** 33 + 16, 128, 256)), FAL_ERR_INVALID, "k_cache: stride[0]"),
    (dict(k_scale_strides=(2 ** 31, 1)), FAL_ERR_INVALID, "k_scale: strides must be"),
    (dict(v_strides=(2 ** 30, 128, 2 ** 22)), FAL_ERR_UNSUPPORTED, "v_cache: row stride"),
    (dict(page_size=1024, max_pages=1, k_strides=(2 ** 32, 128, 2 ** 21 + 16), v_strides=(2 ** 32, 128, 256)), FAL_ERR_UNSUPPORTED,
     "k_cache: a page of 1024 rows"),
    (dict(v_strides=(16384, 128, 112)), FAL_ERR_UNSUPPORTED, "shorter than a row"),
    (dict(k_scale=None), FAL_ERR_INVALID, "k_scale: null pointer"),
    (dict(v_scale=P + 2), FAL_ERR_INVALID, "v_scale: base pointer must be 4-byte aligned"),
    (dict(v_scale_strides=(-2, 1)), FAL_ERR_INVALID, "v_scale: strides must be non-negative"),
    (dict(fp8=0, k_strides=(32768, 128, 256), v_strides=(32768, 128, 256)), FAL_ERR_INVALID, "a 16-bit cache has no scales"),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw,code,msg", BAD_CACHES, ids=lambda x: "")
def test_both_calls_refuse(ext, kw, code, msg, bf16):
    for call in (append, attn):
        rc, err = call(ext, cache(ext, **kw), bf16=bf16)
        assert rc == code and msg in err, (call.__name__, rc, err)


def test_null_cache(ext):
    assert append(ext, None) == (FAL_ERR_INVALID, "cache: null pointer")
    assert attn(ext, None) == (FAL_ERR_INVALID, "cache: null pointer")


def test_append_refuses(ext):
    for kw, c, msg in (
            (dict(), dict(k_strides=(0, 128, 256)), "k_cache: rows overlap"),
            (dict(), dict(v_strides=(16384, 0, 256)), "v_cache: rows overlap"),
            (dict(), dict(v_strides=(16384, 128, 128)), "v_cache: rows overlap"),
            (dict(), dict(k_scale_strides=(0, 1)), "k_scale: entries overlap"),
            (dict(), dict(v_scale_strides=(1, 1)), "v_scale: entries overlap"),
            (dict(), dict(v_scale_strides=(1, 9)), "v_scale: entries overlap"),
            (dict(), dict(v=P), "must not share a cache or scales"),
            (dict(), dict(v_scale=P), "must not share a cache or scales"),
            (dict(k=None), {}, "k: null pointer"),
            (dict(k=P + 2), {}, "k: base pointer must be 16-byte aligned"),
            (dict(q_out=None), {}, "q_out: null pointer"),
            (dict(strides=s3(2048, 100, 1024)), {}, "stride[1]=100 must be"),
            (dict(rotary=24), {}, "rotary_dim must be a multiple of 16 up to head_dim, got 24"),
            (dict(rotary=144), {}, "rotary_dim must be"),
            (dict(rows=255), {}, "255 rows for the 256 positions"),
            (dict(cos=None), {}, "rotary tables: null pointer"),
            (dict(cos_stride=66), {}, "rotary tables: base pointers and rows"),
            (dict(), dict(batch=2 ** 20, total_tokens=2 ** 30, seqlen=2 ** 10, heads_q=512, heads_kv=256,
                          k_strides=(64 * 256 * 128, 128, 256 * 128), v_strides=(64 * 256 * 128, 128, 256 * 128),
                          k_scale_strides=(256, 1), v_scale_strides=(256, 1)), "too large for one launch")):
        rc, err = append(ext, cache(ext, **c), **kw)
        assert rc in (FAL_ERR_INVALID, FAL_ERR_UNSUPPORTED) and msg in err, (msg, rc, err)
    # interleaved pools are no overlap: pages of k and v by turns, scales by head first
    c = cache(ext, total_tokens=0, seqlen=0, k_strides=(2 * 16384, 128, 256), v_strides=(128, 1280, 2560),
              k_scale_strides=(1, 10))
    assert append(ext, c) == (FAL_OK, "")


def test_workspace_size(ext):
    """Nothing for calls that are not recognised, and no more for a hint past the tokens there are."""
    size = lambda **kw: ext._lib.fal_paged_attn_workspace_size(ctypes.byref(cache(ext, **kw)))
    assert ext._lib.fal_paged_attn_workspace_size(None) == 0
    for kw in (dict(heads_q=7), dict(heads_kv=0), dict(page_size=0), dict(max_pages=-1), dict(batch=-1), dict(seqlen=2 ** 40)):
        assert size(**kw) == 0
    assert size(batch=64, seqlen=64, total_tokens=64, cu_seqlens=P, max_pages=1000) == \
        size(batch=64, seqlen=10 ** 9, total_tokens=64, cu_seqlens=P, max_pages=1000)


def test_attention_refuses(ext):
    for kw, msg in ((dict(q=None), "q: null pointer"), (dict(o=P + 8), "o: base pointer"),
                    (dict(strides=s3(2048, 100, 1024)), "stride[1]=100 must be")):
        rc, err = attn(ext, cache(ext), **kw)
        assert rc == FAL_ERR_INVALID and msg in err, (msg, rc, err)
    assert attn(ext, cache(ext, total_tokens=0, seqlen=0)) == (FAL_OK, "")


def test_python_checks():
    from flash_attn_legacy import flash_attn_with_paged_kvcache, paged_kvcache_append
    x = torch.zeros(2, 1, 4, 64)
    table = torch.zeros((2, 1), dtype=torch.int32)
    with pytest.raises(AssertionError, match="float16"):
        paged_kvcache_append(x, x, x, x, table, 0)
    with pytest.raises(AssertionError, match="head_dim must be"):
        flash_attn_with_paged_kvcache(x.half()[..., :48], x, x, table, 0)
    with pytest.raises(AssertionError, match="go together"):
        flash_attn_with_paged_kvcache(x.half(), x, x, table, 0, max_seqlen_q=3)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        flash_attn_with_paged_kvcache(x.half(), x.half(), x.half(), table, 0)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        paged_kvcache_append(x.half(), x.half(), x.half(), x.half(), table, 0)


def test_rotary_tables():
    """Far positions keep their angle: fp32 tables are within a rounding of the 64-bit ones."""
    from flash_attn_legacy import rotary_cos_sin
    cos, sin = rotary_cos_sin(200001, 64, base=500000.0)
    assert cos.shape == sin.shape == (200001, 32) and cos.dtype == torch.float32
    for p, j in ((0, 0), (1, 31), (200000, 0), (123457, 5)):
        a = p * 500000.0 ** (-2 * j / 64)
        # the angle's own rounding in 64 bits, 2^-52 of up to 2e5, and one rounding to 32 bits
        assert abs(float(cos[p, j]) - math.cos(a)) <= 2.0 ** -25 + 1e-10
        assert abs(float(sin[p, j]) - math.sin(a)) <= 2.0 ** -25 + 1e-10
    with pytest.raises(AssertionError, match="even"):
        rotary_cos_sin(4, 33)


def test_oracle_rotation_is_a_rotation():
    from oracle import paged as orc
    x = torch.randn(3, 64, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    angle = torch.rand(5, 16, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    for inter in (False, True):
        y = orc.rotate(x, 2, angle.cos(), angle.sin(), 32, inter)
        pair = (lambda t: torch.complex(t[:, 0:32:2], t[:, 1:32:2])) if inter else (lambda t: torch.complex(t[:, :16], t[:, 16:32]))
        torch.testing.assert_close(pair(y), pair(x) * torch.polar(torch.ones(16, dtype=torch.float64), angle[2]), rtol=1e-12, atol=0)
        assert torch.equal(y[:, 32:], x[:, 32:])


def test_oracle_attention():
    """Against softmax over the gathered rows, with a causal mask aligned at the end."""
    from oracle import paged as orc
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn(6, 16, 2, 32, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.tensor([[4, 0, 5], [2, 3, 1]])
    q = torch.randn(5, 4, 32, generator=g, dtype=torch.float64)
    o, lse, mass, spread, qk = orc.attend(q, kc, vc, table, [40, 3], [0, 3, 5], 0.3, True)
    for b, t0, n, m in ((0, 0, 3, 40), (1, 3, 2, 3)):
        k, v = (c[table[b]].reshape(-1, 2, 32)[:m] for c in (kc, vc))
        for i in range(n):
            for h in range(4):
                s = 0.3 * (k[:m - n + i + 1, h // 2] @ q[t0 + i, h])
                p = torch.softmax(s, 0)
                torch.testing.assert_close(o[t0 + i, h], p @ v[:len(s), h // 2], rtol=1e-12, atol=1e-14)
                assert abs(float(lse[t0 + i, h]) - math.log(float(s.exp().sum()))) < 1e-12
