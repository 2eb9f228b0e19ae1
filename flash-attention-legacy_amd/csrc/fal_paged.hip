// Paged KV cache for gfx950: rotation and append of new rows, and attention of one or more new
// tokens per sequence to the cache.  No counterpart in the reference, whose caches are
// contiguous 16-bit tensors read by eager PyTorch (flash_attn_legacy/integrations.py:77-98).
//
// 8-bit caches hold e4m3 codes with one fp32 scale per (page, KV head), K and V apart.  The
// scales that the append chooses are powers of two: a floating-point format has the same
// relative precision wherever its scale puts it, multiplying by the scale is exact, and when a
// later token raises a page's scale the older codes keep their mantissas (only what falls
// below e4m3's smallest normal is rounded again).
#include <type_traits>

#include "fal_kernels.h"

namespace fal {

constexpr float kE4m3Max = 448.f;   // largest finite value of e4m3
constexpr int kMinScaleExp = -126;  // 2^-126 and its reciprocal are normal fp32 numbers

// Token range of sequence b: rows off .. off + len of the packed tokens, or of batch entry b.
__device__ __forceinline__ void token_range(const PagedCache& c, int b, int& off, int& len) {
  off = 0, len = c.n;
  if (c.cu) seg_bounds(c.cu, b, c.total, off, len);
}

// Sequence and place in it of token t (row of the packed tokens, or of [B, n]); false for a
// row outside every sequence.
__device__ __forceinline__ bool token_place(const PagedCache& c, int t, int& b, int& i) {
  if (!c.cu) {
    b = t / c.n;
    i = t - b * c.n;
    return true;
  }
  int lo = 0, hi = c.B;   // the last b with cu[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c.cu[mid] <= t) lo = mid; else hi = mid;
  }
  int len;
  seg_bounds(c.cu, lo, c.total, i, len);
  b = lo;
  i = t - i;
  return i >= 0 && i < len;
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------

// Two chunks of eight elements of a row, rotated where the rotation covers them.  Unit u of a
// row of D elements: in half-split pairs (x_j, x_{j + r/2}) the chunks u and u + r/16 for
// u < r/16, and otherwise the chunks 2u and 2u + 1, which hold the interleaved pairs; both use
// the angles 8u .. 8u + 7.  The products and the sum are rounded one by one (no contraction),
// so the values do not depend on the compiler's choice.
template <class T>
__device__ __forceinline__ void load_unit(const T* row, int u, int rotary, int interleaved, const float* cs,
                                          const float* sn, int& ca, int& cb, float (&y)[16]) {
#pragma clang fp contract(off)
  const bool rot = u * 16 < rotary;
  const bool halves = rot && !interleaved;
  ca = halves ? u : 2 * u;
  cb = halves ? u + rotary / 16 : 2 * u + 1;
  const vec8<T> a = ld8(row + ca * 8), b = ld8(row + cb * 8);
  if (!rot) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)a[j], y[8 + j] = (float)b[j];
    return;
  }
  f32x4 c[2], s[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    c[j] = *reinterpret_cast<const f32x4*>(cs + u * 8 + 4 * j);
    s[j] = *reinterpret_cast<const f32x4*>(sn + u * 8 + 4 * j);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float cj = c[j / 4][j % 4], sj = s[j / 4][j % 4];
    // pair j: elements (j, 8 + j) of the two chunks, or (2j, 2j + 1) of the sixteen
    const float x1 = halves ? (float)a[j] : (float)(j < 4 ? a[2 * j & 7] : b[2 * j & 7]);
    const float x2 = halves ? (float)b[j] : (float)(j < 4 ? a[(2 * j + 1) & 7] : b[(2 * j + 1) & 7]);
    const float p1 = x1 * cj, p2 = x2 * sj, p3 = x2 * cj, p4 = x1 * sj;
    const float y1 = p1 - p2, y2 = p3 + p4;
    if (halves) y[j] = y1, y[8 + j] = y2;
    else y[2 * j] = y1, y[2 * j + 1] = y2;
  }
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;   // NaN and infinity: 0
}

// The smallest 2^e, e >= -126, with amax <= 448 * 2^e (448 = 0.875 * 2^9).
__device__ __forceinline__ float page_scale(float amax) {
  int e;
  const float m = frexpf(amax, &e);
  e = amax > 0.f ? e - 9 + (m > 0.875f ? 1 : 0) : kMinScaleExp;
  return ldexpf(1.f, max(e, kMinScaleExp));
}

// Saturated to +-448 (infinities too; NaN stays NaN)
__device__ __forceinline__ float e4m3_sat(float x) {
  return x != x ? x : fminf(fmaxf(x, -kE4m3Max), kE4m3Max);
}
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_sat(a), e4m3_sat(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_sat(c), e4m3_sat(d), r, true);
}
__device__ __forceinline__ void e4m3_unpack4(uint32_t x, float (&y)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  y[0] = lo[0], y[1] = lo[1], y[2] = hi[0], y[3] = hi[1];
}

// 8 values of a chunk to the cache row
template <class T>
__device__ __forceinline__ void put_chunk(T* row, int chunk, const float* y) {
  vec8<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)y[j];
  st_u4(row + chunk * 8, __builtin_bit_cast(u32x4, r));
}
__device__ __forceinline__ void put_chunk8(uint8_t* row, int chunk, const float* y, float inv) {
  u32x2 r;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    r[j] = e4m3_pack4(y[4 * j] * inv, y[4 * j + 1] * inv, y[4 * j + 2] * inv, y[4 * j + 3] * inv);
  *reinterpret_cast<u32x2*>(row + chunk * 8) = r;
}

// Blocks below `store_blocks`: one touched page of one sequence, KV head and side (K or V).
// Such a block owns the page's rows and scale for its head, so nothing is atomic and the
// result does not depend on timing.  The others rotate queries, one unit per thread.
constexpr int kAppendHold = 4;   // units per thread kept in registers between the two passes

template <class T, bool FP8, int D>
__global__ void __launch_bounds__(256)
paged_append_kernel(PagedAppendParams p, int store_blocks) {
  constexpr int UPR = D / 16;   // units per row
  const PagedCache& c = p.c;
  const int nt = blockDim.x, tid = threadIdx.x;
  if ((int)blockIdx.x >= store_blocks) {
    const int64_t unit = (int64_t)((int)blockIdx.x - store_blocks) * nt + tid;
    const int u = (int)(unit % UPR);
    const int64_t row = unit / UPR;
    if (row >= (int64_t)c.total * c.Hq) return;
    const int t = (int)(row / c.Hq), h = (int)(row % c.Hq);
    int b, i;
    const bool in = token_place(c, t, b, i);
    const int64_t pos = in ? (int64_t)max(c.seqlens[b], 0) + i : c.capacity;
    T* out = (T*)p.q_out + (c.cu ? t * p.qo_ss : b * p.qo_sb + i * p.qo_ss) + h * p.qo_sh;
    if (pos >= c.capacity) {   // outside every sequence, or past the table
      st_u4(out + u * 16, u32x4{0, 0, 0, 0});
      st_u4(out + u * 16 + 8, u32x4{0, 0, 0, 0});
      return;
    }
    const T* in_row = (const T*)p.q + (c.cu ? t * p.q_ss : b * p.q_sb + i * p.q_ss) + h * p.q_sh;
    int ca, cb;
    float y[16];
    load_unit(in_row, u, p.rotary, p.interleaved, p.cos + pos * p.cos_ss, p.sin + pos * p.sin_ss, ca, cb, y);
    put_chunk(out, ca, y);
    put_chunk(out, cb, y + 8);
    return;
  }

  __shared__ float wave_max[4];
  const int h = blockIdx.x % c.Hkv;
  int rest = blockIdx.x / c.Hkv;
  const bool is_v = rest & 1;
  rest >>= 1;
  const int b = rest / p.pages_per_seq;
  int off, len;
  token_range(c, b, off, len);
  const int L = max(c.seqlens[b], 0);
  const int64_t end = min((int64_t)L + len, (int64_t)c.capacity);   // rows after the append
  const T* src = is_v ? (const T*)p.v + (c.cu ? off * p.v_ss : b * p.v_sb) + h * p.v_sh
                      : (const T*)p.k + (c.cu ? off * p.k_ss : b * p.k_sb) + h * p.k_sh;
  const int64_t src_ss = is_v ? p.v_ss : p.k_ss;
  const int64_t dst_ss = is_v ? c.v_ss : c.k_ss;
  const int rotary = is_v ? 0 : p.rotary;
  for (int64_t page = L / c.page_size + rest % p.pages_per_seq; page * c.page_size < end; page += p.pages_per_seq) {
    const int pid = c.table[b * c.table_sb + page];
    if (pid < 0 || pid >= c.num_pages) continue;
    const int64_t first = page * c.page_size;
    const int r0 = (int)(max((int64_t)L, first) - first);                // first new row of the page
    const int rows = (int)(min(end, first + c.page_size) - first) - r0;
    if (rows <= 0) continue;
    const int i0 = (int)(first + r0 - L);                                // its token
    const int total = rows * UPR;
    auto load = [&](int e, int& r, int& ca, int& cb, float (&y)[16]) {
      r = e / UPR;
      const int64_t pos = first + r0 + r;
      load_unit(src + (int64_t)(i0 + r) * src_ss, e % UPR, rotary, p.interleaved, p.cos + pos * p.cos_ss,
                p.sin + pos * p.sin_ss, ca, cb, y);
    };
    if constexpr (!FP8) {
      T* dst = (is_v ? (T*)c.v + pid * c.v_sp + h * c.v_sh : (T*)c.k + pid * c.k_sp + h * c.k_sh) + r0 * dst_ss;
      for (int e = tid; e < total; e += nt) {
        int r, ca, cb;
        float y[16];
        load(e, r, ca, cb, y);
        put_chunk(dst + r * dst_ss, ca, y);
        put_chunk(dst + r * dst_ss, cb, y + 8);
      }
    } else {
      uint8_t* base = is_v ? (uint8_t*)c.v + pid * c.v_sp + h * c.v_sh : (uint8_t*)c.k + pid * c.k_sp + h * c.k_sh;
      uint8_t* dst = base + r0 * dst_ss;
      float* sp = is_v ? c.v_scale + pid * c.vs_sp + h * c.vs_sh : c.k_scale + pid * c.ks_sp + h * c.ks_sh;
      const float old = r0 > 0 ? *sp : 0.f;   // filled from its first row on: the old scale is another sequence's
      float held[kAppendHold][16];
      float amax = 0.f;
#pragma unroll
      for (int q = 0; q < kAppendHold; ++q) {
        const int e = tid + q * nt;
        if (e < total) {
          int r, ca, cb;
          load(e, r, ca, cb, held[q]);
#pragma unroll
          for (int j = 0; j < 16; ++j) amax = fmaxf(amax, finite_abs(held[q][j]));
        }
      }
      for (int e = tid + kAppendHold * nt; e < total; e += nt) {
        int r, ca, cb;
        float y[16];
        load(e, r, ca, cb, y);
#pragma unroll
        for (int j = 0; j < 16; ++j) amax = fmaxf(amax, finite_abs(y[j]));
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
      __syncthreads();   // wave_max of the previous page has been read
      if ((tid & 63) == 0) wave_max[tid >> 6] = amax;
      __syncthreads();
      for (int w = 0; w < (nt + 63) / 64; ++w) amax = fmaxf(amax, wave_max[w]);
      const float scale = fmaxf(old, page_scale(amax));   // (an old NaN counts as none)
      const float inv = 1.f / scale;
      if (tid == 0) *sp = scale;
      if (r0 > 0 && scale > old) {   // the rows before the new ones, in the new units
        const float ratio = old * inv;
        for (int e = tid; e < r0 * (D / 16); e += nt) {
          u32x4* at = reinterpret_cast<u32x4*>(base + (int64_t)(e / (D / 16)) * dst_ss + (e % (D / 16)) * 16);
          u32x4 x = *at;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float y[4];
            e4m3_unpack4(x[j], y);
            x[j] = e4m3_pack4(y[0] * ratio, y[1] * ratio, y[2] * ratio, y[3] * ratio);
          }
          *at = x;
        }
      }
#pragma unroll
      for (int q = 0; q < kAppendHold; ++q) {
        const int e = tid + q * nt;
        if (e < total) {
          const int u = e % UPR;
          const bool halves = u * 16 < rotary && !p.interleaved;
          uint8_t* row = dst + (int64_t)(e / UPR) * dst_ss;
          put_chunk8(row, halves ? u : 2 * u, held[q], inv);
          put_chunk8(row, halves ? u + rotary / 16 : 2 * u + 1, held[q] + 8, inv);
        }
      }
      for (int e = tid + kAppendHold * nt; e < total; e += nt) {
        int r, ca, cb;
        float y[16];
        load(e, r, ca, cb, y);
        put_chunk8(dst + r * dst_ss, ca, y, inv);
        put_chunk8(dst + r * dst_ss, cb, y + 8, inv);
      }
    }
  }
}

template <class T, bool FP8, int D>
static hipError_t launch_append_t(const PagedAppendParams& p, hipStream_t st) {
  const PagedCache& c = p.c;
  // threads: a page's new rows in one unit each, up to four waves
  const int rows = c.n < c.page_size ? c.n : c.page_size;
  int nt = (rows * (D / 16) + 63) / 64 * 64;
  nt = nt > 256 ? 256 : nt;
  const int64_t store = (int64_t)c.B * p.pages_per_seq * 2 * c.Hkv;
  const int64_t query = p.q ? ((int64_t)c.total * c.Hq * (D / 16) + nt - 1) / nt : 0;
  if (store + query > 0x7fffffff) return hipErrorInvalidValue;
  if (store + query == 0) return hipSuccess;
  hipLaunchKernelGGL((paged_append_kernel<T, FP8, D>), dim3((unsigned)(store + query)), dim3(nt), 0, st, p, (int)store);
  return hipGetLastError();
}

template <int D>
static hipError_t launch_append_d(const PagedAppendParams& p, hipStream_t st) {
  if (p.c.fp8) return p.c.bf16 ? launch_append_t<bf16_t, true, D>(p, st) : launch_append_t<half_t, true, D>(p, st);
  return p.c.bf16 ? launch_append_t<bf16_t, false, D>(p, st) : launch_append_t<half_t, false, D>(p, st);
}

hipError_t launch_paged_append(const PagedAppendParams& p, int d, hipStream_t st) {
  switch (d) {
    case 32: return launch_append_d<32>(p, st);
    case 64: return launch_append_d<64>(p, st);
    case 96: return launch_append_d<96>(p, st);
    case 128: return launch_append_d<128>(p, st);
    case 256: return launch_append_d<256>(p, st);
    default: return hipErrorInvalidValue;
  }
}

// ---------------------------------------------------------------------------
// Attention: one workgroup per (token, query head), one wave per four rows
// ---------------------------------------------------------------------------
template <class T, bool FP8>
__device__ __forceinline__ float cache_elem(const void* row, int e) {
  if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)row)[e], 0);
  else return (float)((const T*)row)[e];
}

template <class T, bool FP8, int D>
__global__ void __launch_bounds__(256)
paged_attn_simple_kernel(PagedAttnParams p) {
  const PagedCache& c = p.c;
  constexpr int CB = FP8 ? 1 : 2, DJ = (D + 63) / 64;
  __shared__ float m_s[4], l_s[4], o_s[4][D];
  const int t = blockIdx.x / c.Hq, h = blockIdx.x % c.Hq, hk = h / (c.Hq / c.Hkv);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int b = 0, i = 0, off = 0, len = 0, end = 0;
  if (token_place(c, t, b, i)) {
    token_range(c, b, off, len);
    const int L = min(max(c.seqlens[b], 0), c.capacity);
    end = p.causal ? max(L - len + i + 1, 0) : L;
  }
  const T* qrow = (const T*)p.q + (c.cu ? t * p.q_ss : b * p.q_sb + i * p.q_ss) + h * p.q_sh;
  T* orow = (T*)p.o + (c.cu ? t * p.o_ss : b * p.o_sb + i * p.o_ss) + h * p.o_sh;
  float q[DJ], o[DJ];
#pragma unroll
  for (int j = 0; j < DJ; ++j) {
    const int e = lane + 64 * j;
    q[j] = e < D ? (float)qrow[e] * (p.negate_q ? -p.scale_log2 : p.scale_log2) : 0.f;
    o[j] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int r = w; r < end; r += 4) {
    const int pid = c.table[b * c.table_sb + r / c.page_size];
    if (pid < 0 || pid >= c.num_pages) continue;
    const char* k = (const char*)c.k + (pid * c.k_sp + hk * c.k_sh + (r % c.page_size) * c.k_ss) * CB;
    const char* v = (const char*)c.v + (pid * c.v_sp + hk * c.v_sh + (r % c.page_size) * c.v_ss) * CB;
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < DJ; ++j)
      if (lane + 64 * j < D) x = fmaf(q[j], cache_elem<T, FP8>(k, lane + 64 * j), x);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s);
    if (FP8) x *= c.k_scale[pid * c.ks_sp + hk * c.ks_sh];
    const float mn = fmaxf(m, x), use = mn == -INFINITY ? 0.f : mn;
    const float a = fast_exp2(m - use), e = fast_exp2(x - use);
    m = mn;
    l = l * a + e;
    const float ev = FP8 ? e * c.v_scale[pid * c.vs_sp + hk * c.vs_sh] : e;
#pragma unroll
    for (int j = 0; j < DJ; ++j)
      if (lane + 64 * j < D) o[j] = fmaf(ev, cache_elem<T, FP8>(v, lane + 64 * j), o[j] * a);
  }
  if (lane == 0) m_s[w] = m, l_s[w] = l;
#pragma unroll
  for (int j = 0; j < DJ; ++j)
    if (lane + 64 * j < D) o_s[w][lane + 64 * j] = o[j];
  __syncthreads();
  if (w) return;
  const float M = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
  const float use = M == -INFINITY ? 0.f : M;
  float total = 0.f;
  for (int x = 0; x < 4; ++x) total += l_s[x] * fast_exp2(m_s[x] - use);
  const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int j = 0; j < DJ; ++j) {
    const int e = lane + 64 * j;
    float acc = 0.f;
    if (e < D) {
      for (int x = 0; x < 4; ++x) acc += o_s[x][e] * fast_exp2(m_s[x] - use);
      orow[e] = (T)(acc * inv);
    }
  }
  if (p.lse && lane == 0) p.lse[(int64_t)t * c.Hq + h] = total > 0.f ? (use + fast_log2(total)) * kLn2 : -INFINITY;
}

template <int D>
static hipError_t launch_attn_d(const PagedAttnParams& p, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)p.c.total * p.c.Hq));
  if (p.c.fp8) {
    if (p.c.bf16) hipLaunchKernelGGL((paged_attn_simple_kernel<bf16_t, true, D>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attn_simple_kernel<half_t, true, D>), grid, dim3(256), 0, st, p);
  } else {
    if (p.c.bf16) hipLaunchKernelGGL((paged_attn_simple_kernel<bf16_t, false, D>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attn_simple_kernel<half_t, false, D>), grid, dim3(256), 0, st, p);
  }
  return hipGetLastError();
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int d, hipStream_t st) {
  switch (d) {
    case 32: return launch_attn_d<32>(p, st);
    case 64: return launch_attn_d<64>(p, st);
    case 96: return launch_attn_d<96>(p, st);
    case 128: return launch_attn_d<128>(p, st);
    case 256: return launch_attn_d<256>(p, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fal
