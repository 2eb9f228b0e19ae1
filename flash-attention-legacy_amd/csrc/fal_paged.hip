// Paged KV cache for gfx950: rotation and append of new rows, and attention of one or more new
// tokens per sequence to the cache.  No counterpart in the reference, whose caches are
// contiguous 16-bit tensors read by eager PyTorch (flash_attn_legacy/integrations.py:77-98).
//
// 8-bit caches hold e4m3 codes with one fp32 scale per (page, KV head), K and V apart.  The
// scales that the append chooses are powers of two: a floating-point format has the same
// relative precision wherever its scale puts it, multiplying by the scale is exact, and when a
// later token raises a page's scale the older codes keep their mantissas (only what falls
// below e4m3's smallest normal is rounded again).
#include <algorithm>
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

__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); }

// Inclusive sum over the wave's lanes (row shifts, then the rows' last lanes broadcast)
__device__ __forceinline__ int lanes_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast:31
  return x;
}

// Batches are searched by blocks of 64 sequences, one per lane, four blocks read at once: large
// batches cost one round trip to memory in 256 sequences.
constexpr int kBlocks = 4;

// Which of `cnt`'s lanes' items, in the lanes' order, the r-th is: the lane; r becomes its place
// among that lane's.  `sum`: lanes_scan(cnt).
__device__ __forceinline__ int lane_of_item(uint32_t cnt, uint32_t sum, uint32_t& r) {
  const auto past = __ballot(sum > r);
  const int at = past ? __builtin_ctzll(past) : 0;
  r -= lane_of(sum, at) - lane_of(cnt, at);
  return at;
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------

enum { kNoRotation, kHalves, kInterleaved };

// The chunks (eight elements) of unit u of a row: chunks u and u + r/16 of the half-split pairs
// (x_j, x_{j + r/2}) for u < r/16, and otherwise 2u and 2u + 1, which hold the interleaved pairs.
// A unit's pairs use the angles 8u .. 8u + 7 either way.
template <int MODE>
__device__ __forceinline__ void unit_chunks(int u, int rotary, int& ca, int& cb) {
  const bool halves = MODE == kHalves && u * 16 < rotary;
  ca = halves ? u : 2 * u;
  cb = halves ? u + rotary / 16 : 2 * u + 1;
}
struct Angles {
  f32x4 c[2], s[2];
};
template <int MODE>
__device__ __forceinline__ Angles unit_angles(int u, int rotary, const float* cs, const float* sn) {
  Angles t;
  if (MODE == kNoRotation || u * 16 >= rotary) return t;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    t.c[j] = *reinterpret_cast<const f32x4*>(cs + u * 8 + 4 * j);
    t.s[j] = *reinterpret_cast<const f32x4*>(sn + u * 8 + 4 * j);
  }
  return t;
}

// The unit's sixteen values, rotated where the rotation covers them.  The products and the sum
// are rounded one by one (no contraction), so the values do not depend on the compiler's choice.
template <int MODE, class T, int D>
__device__ __forceinline__ void rotate_unit(vec8<T> a, vec8<T> b, int u, int rotary, const Angles& t, float (&y)[16]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = (float)a[j], y[8 + j] = (float)b[j];
  if (MODE == kNoRotation || (rotary < D && u * 16 >= rotary)) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i1 = MODE == kHalves ? j : 2 * j, i2 = MODE == kHalves ? 8 + j : 2 * j + 1;
    const float cj = t.c[j / 4][j % 4], sj = t.s[j / 4][j % 4], x1 = y[i1], x2 = y[i2];
    const float p1 = x1 * cj, p2 = x2 * sj, p3 = x2 * cj, p4 = x1 * sj;
    y[i1] = p1 - p2, y[i2] = p3 + p4;
  }
}

// The smallest 2^e, e >= -126, with amax <= 448 * 2^e (448 = 0.875 * 2^9).
__device__ __forceinline__ float page_scale(float amax) {
  int e;
  const float m = frexpf(amax, &e);
  e = amax > 0.f ? e - 9 + (m > 0.875f ? 1 : 0) : kMinScaleExp;
  return ldexpf(1.f, max(e, kMinScaleExp));
}

// Values of at most 448 in magnitude (or NaN) as codes
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ void e4m3_unpack4(uint32_t x, float (&y)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  y[0] = lo[0], y[1] = lo[1], y[2] = hi[0], y[3] = hi[1];
}

// 8 values of a chunk to a 16-bit row, or as codes in units of 1 / inv
template <class T>
__device__ __forceinline__ void put_chunk(T* row, int chunk, const float* y) {
  vec8<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)y[j];
  st_u4(row + chunk * 8, __builtin_bit_cast(u32x4, r));
}
__device__ __forceinline__ void put_codes(uint8_t* row, int chunk, const float* y, float inv) {
  u32x2 r;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    r[j] = e4m3_pack4(y[4 * j] * inv, y[4 * j + 1] * inv, y[4 * j + 2] * inv, y[4 * j + 3] * inv);
  *reinterpret_cast<u32x2*>(row + chunk * 8) = r;
}
// y * inv, infinities as the largest code (NaN stays)
__device__ __forceinline__ void scale_saturated(float (&y)[16], float inv) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float x = y[j] * inv;
    y[j] = x != x ? x : fminf(fmaxf(x, -kE4m3Max), kE4m3Max);
  }
}

// Rows to rows: units of one token and position in the row for kRowHeads heads, whose angles are
// read once.  Queries go to q_out; with a 16-bit cache keys and values go to their pages.
constexpr int kRowHeads = 4;

template <int MODE, class T, int D>
__device__ __forceinline__ void copy_heads(const T* src, int64_t src_sh, T* dst, int64_t dst_sh, int heads, int u,
                                           int rotary, const float* cs, const float* sn) {
  int ca, cb;
  unit_chunks<MODE>(u, rotary, ca, cb);
  vec8<T> a[kRowHeads], b[kRowHeads];
#pragma unroll
  for (int i = 0; i < kRowHeads; ++i)
    if (i < heads) a[i] = ld8(src + i * src_sh + ca * 8), b[i] = ld8(src + i * src_sh + cb * 8);
  const Angles t = unit_angles<MODE>(u, rotary, cs, sn);
#pragma unroll
  for (int i = 0; i < kRowHeads; ++i)
    if (i < heads) {
      float y[16];
      rotate_unit<MODE, T, D>(a[i], b[i], u, rotary, t, y);
      put_chunk(dst + i * dst_sh, ca, y);
      put_chunk(dst + i * dst_sh, cb, y + 8);
    }
}

template <class T, int D>
__device__ void append_rows(const PagedAppendParams& p, int64_t item) {
  constexpr int UPR = D / 16;
  const PagedCache& c = p.c;
  const int u = (int)(item % UPR);
  item /= UPR;
  const int group = (int)(item % p.row_groups);
  const int64_t t = item / p.row_groups;
  if (t >= c.total) return;
  int b, i;
  const bool in = token_place(c, (int)t, b, i);
  const int64_t pos = in ? (int64_t)max(c.seqlens[b], 0) + i : c.capacity;
  const int qg = p.q ? cdiv(c.Hq, kRowHeads) : 0, kg = cdiv(c.Hkv, kRowHeads);
  if (group < qg) {
    const int h = group * kRowHeads, n = min(kRowHeads, c.Hq - h);
    T* out = (T*)p.q_out + (c.cu ? t * p.qo_ss : b * p.qo_sb + i * p.qo_ss) + h * p.qo_sh;
    if (pos >= c.capacity) {   // outside every sequence, or past the table
      for (int x = 0; x < n; ++x) {
        st_u4(out + x * p.qo_sh + u * 16, u32x4{0, 0, 0, 0});
        st_u4(out + x * p.qo_sh + u * 16 + 8, u32x4{0, 0, 0, 0});
      }
      return;
    }
    const T* q = (const T*)p.q + (c.cu ? t * p.q_ss : b * p.q_sb + i * p.q_ss) + h * p.q_sh;
    const float *cs = p.cos + pos * p.cos_ss, *sn = p.sin + pos * p.sin_ss;
    if (!p.rotary) copy_heads<kNoRotation, T, D>(q, p.q_sh, out, p.qo_sh, n, u, 0, cs, sn);
    else if (p.interleaved) copy_heads<kInterleaved, T, D>(q, p.q_sh, out, p.qo_sh, n, u, p.rotary, cs, sn);
    else copy_heads<kHalves, T, D>(q, p.q_sh, out, p.qo_sh, n, u, p.rotary, cs, sn);
    return;
  }
  if (pos >= c.capacity) return;
  const int page = (int)(pos / c.page_size), slot = (int)(pos - (int64_t)page * c.page_size);
  const int pid = c.table[b * c.table_sb + page];
  if (pid < 0 || pid >= c.num_pages) return;
  const bool is_v = group - qg >= kg;
  const int h = (is_v ? group - qg - kg : group - qg) * kRowHeads, n = min(kRowHeads, c.Hkv - h);
  if (is_v) {
    const T* v = (const T*)p.v + (c.cu ? t * p.v_ss : b * p.v_sb + i * p.v_ss) + h * p.v_sh;
    T* to = (T*)c.v + pid * c.v_sp + h * c.v_sh + slot * c.v_ss;
    copy_heads<kNoRotation, T, D>(v, p.v_sh, to, c.v_sh, n, u, 0, nullptr, nullptr);
    return;
  }
  const T* k = (const T*)p.k + (c.cu ? t * p.k_ss : b * p.k_sb + i * p.k_ss) + h * p.k_sh;
  T* to = (T*)c.k + pid * c.k_sp + h * c.k_sh + slot * c.k_ss;
  const float *cs = p.cos + pos * p.cos_ss, *sn = p.sin + pos * p.sin_ss;
  if (!p.rotary) copy_heads<kNoRotation, T, D>(k, p.k_sh, to, c.k_sh, n, u, 0, cs, sn);
  else if (p.interleaved) copy_heads<kInterleaved, T, D>(k, p.k_sh, to, c.k_sh, n, u, p.rotary, cs, sn);
  else copy_heads<kHalves, T, D>(k, p.k_sh, to, c.k_sh, n, u, p.rotary, cs, sn);
}

// Rows to codes: one touched page of one sequence and KV head, K or V, per workgroup.  It owns
// the page's rows and scale for its head, so nothing is atomic and the result does not depend on
// timing.  Two passes, for the largest magnitude and for the codes; each thread keeps its first
// units in registers between them and reads the others again (from L2).
constexpr int kAppendHold = 2, kAppendThreads = 512;

template <int MODE, class T, int D>
__device__ void append_codes(const PagedAppendParams& p, int b, int h, int nth, const T* src, int64_t src_ss,
                             uint8_t* cache, int64_t dst_sp, int64_t dst_ss, float* scales, int64_t scale_sp, float* wave_max) {
  constexpr int UPR = D / 16;   // units per row
  const PagedCache& c = p.c;
  const int nt = blockDim.x, tid = threadIdx.x;
  int off, len;
  token_range(c, b, off, len);
  const int L = max(c.seqlens[b], 0);
  const int64_t end = min((int64_t)L + len, (int64_t)c.capacity);   // rows after the append
  if (c.cu) src += off * src_ss;
  const int64_t page = L / c.page_size + nth;
  if (page * c.page_size >= end) return;
  const int pid = c.table[b * c.table_sb + page];
  if (pid < 0 || pid >= c.num_pages) return;
  const int64_t first = page * c.page_size;
  const int r0 = (int)(max((int64_t)L, first) - first);                // first new row of the page
  const int rows = (int)(min(end, first + c.page_size) - first) - r0;
  if (rows <= 0) return;
  const int64_t i0 = first + r0 - L;                                   // its token
  const int total = rows * UPR;
  uint8_t* base = cache + pid * dst_sp;
  float* sp = scales + pid * scale_sp;
  const float old = r0 > 0 ? *sp : 0.f;   // filled from its first row on: the old scale is another sequence's
  auto load = [&](int e, float (&y)[16]) {
    const int r = e / UPR, u = e % UPR;
    int ca, cb;
    unit_chunks<MODE>(u, p.rotary, ca, cb);
    const T* row = src + (i0 + r) * src_ss;
    const int64_t pos = first + r0 + r;
    const vec8<T> a = ld8(row + ca * 8), b8 = ld8(row + cb * 8);
    const Angles t = unit_angles<MODE>(u, p.rotary, p.cos + pos * p.cos_ss, p.sin + pos * p.sin_ss);
    rotate_unit<MODE, T, D>(a, b8, u, p.rotary, t, y);
  };
  auto store = [&](int e, const float (&y)[16], float inv) {
    const int r = e / UPR, u = e % UPR;
    int ca, cb;
    unit_chunks<MODE>(u, p.rotary, ca, cb);
    uint8_t* row = base + (r0 + r) * dst_ss;
    put_codes(row, ca, y, inv);
    put_codes(row, cb, y + 8, inv);
  };
  float held[kAppendHold][16];
  float amax = 0.f;   // (fmaxf passes over NaN)
#pragma unroll
  for (int q = 0; q < kAppendHold; ++q) {
    const int e = tid + q * nt;
    if (e < total) {
      load(e, held[q]);
#pragma unroll
      for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(held[q][j]));
    }
  }
  for (int e = tid + kAppendHold * nt; e < total; e += nt) {
    float y[16];
    load(e, y);
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(y[j]));
  }
  auto of_all = [&](float x) {   // the largest of the workgroup's threads
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    __syncthreads();   // what wave_max held has been read
    if ((tid & 63) == 0) wave_max[tid >> 6] = x;
    __syncthreads();
    for (int w = 0; w < (nt + 63) / 64; ++w) x = fmaxf(x, wave_max[w]);
    return x;
  };
  amax = of_all(amax);
  const bool infinite = amax == INFINITY;
  if (infinite) {   // once more, of the finite ones
    amax = 0.f;
    for (int e = tid; e < total; e += nt) {
      float y[16];
      load(e, y);
#pragma unroll
      for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(y[j]) < INFINITY ? fabsf(y[j]) : 0.f);
    }
    amax = of_all(amax);
  }
  const float scale = fmaxf(old, page_scale(amax));   // (an old NaN counts as none)
  const float inv = 1.f / scale;
  if (tid == 0) *sp = scale;
  if (r0 > 0 && scale > old) {   // the rows before the new ones, in the new units
    const float ratio = old * inv;
    for (int e = tid; e < r0 * UPR; e += nt) {
      u32x4* at = reinterpret_cast<u32x4*>(base + (int64_t)(e / UPR) * dst_ss + (e % UPR) * 16);
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
      if (infinite) scale_saturated(held[q], inv);
      store(e, held[q], infinite ? 1.f : inv);
    }
  }
  for (int e = tid + kAppendHold * nt; e < total; e += nt) {
    float y[16];
    load(e, y);
    if (infinite) scale_saturated(y, inv);
    store(e, y, infinite ? 1.f : inv);
  }
}

// Page `item` of all that packed tokens touch, sequence by sequence: the sequence and which of
// its pages; false past the last.
__device__ __forceinline__ bool touched_page(const PagedCache& c, int64_t item, int& b, int& nth) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < c.B; base += 64 * kBlocks) {
    uint32_t n[kBlocks], sum[kBlocks];
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      const int s = base + 64 * k + lane;
      n[k] = 0;
      if (s < c.B) {
        int off, len;
        seg_bounds(c.cu, s, c.total, off, len);
        const int L = max(c.seqlens[s], 0), end = (int)min((int64_t)L + len, (int64_t)c.capacity);
        if (end > L) n[k] = (uint32_t)(end - 1) / (uint32_t)c.page_size - (uint32_t)L / (uint32_t)c.page_size + 1;
      }
    }
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      if (base + 64 * k >= c.B) return false;
      sum[k] = (uint32_t)lanes_scan((int)n[k]);
      const uint32_t all = lane_of(sum[k], 63);
      if (item < all) {
        uint32_t r = (uint32_t)item;
        b = base + 64 * k + lane_of_item(n[k], sum[k], r);
        nth = (int)r;
        return nth >= 0;   // (less only if offsets are not monotone and the pages' sum passed 32 bits)
      }
      item -= all;
    }
  }
  return false;
}

// Blocks below `page_blocks` write codes, the others rows.  A workgroup takes one page, of packed
// tokens more if they touch more than the host counted on.  (A workgroup per sequence and page of
// the longest one's: 255 tokens and a prompt of 8192, 916 us; by touched pages 77.)
template <class T, bool FP8, int D>
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(PagedAppendParams p, int page_blocks) {
  const PagedCache& c = p.c;
  if ((int)blockIdx.x >= page_blocks) {
    append_rows<T, D>(p, (int64_t)((int)blockIdx.x - page_blocks) * blockDim.x + threadIdx.x);
    return;
  }
  if constexpr (FP8) {
    __shared__ float wave_max[kAppendThreads / 64];
    const int h = blockIdx.x % c.Hkv;
    int rest = blockIdx.x / c.Hkv;
    const bool is_v = rest & 1;
    rest >>= 1;
    int64_t item = rest;
    do {
      int b = rest / p.pages_per_seq, nth = rest % p.pages_per_seq;
      if (c.cu && !touched_page(c, item, b, nth)) return;
      if (is_v) {
        append_codes<kNoRotation, T, D>(p, b, h, nth, (const T*)p.v + (c.cu ? 0 : b * p.v_sb) + h * p.v_sh, p.v_ss,
                                        (uint8_t*)c.v + h * c.v_sh, c.v_sp, c.v_ss, c.v_scale + h * c.vs_sh, c.vs_sp, wave_max);
        continue;
      }
      const T* k = (const T*)p.k + (c.cu ? 0 : b * p.k_sb) + h * p.k_sh;
      uint8_t* to = (uint8_t*)c.k + h * c.k_sh;
      float* sc = c.k_scale + h * c.ks_sh;
      if (!p.rotary) append_codes<kNoRotation, T, D>(p, b, h, nth, k, p.k_ss, to, c.k_sp, c.k_ss, sc, c.ks_sp, wave_max);
      else if (p.interleaved) append_codes<kInterleaved, T, D>(p, b, h, nth, k, p.k_ss, to, c.k_sp, c.k_ss, sc, c.ks_sp, wave_max);
      else append_codes<kHalves, T, D>(p, b, h, nth, k, p.k_ss, to, c.k_sp, c.k_ss, sc, c.ks_sp, wave_max);
    } while (c.cu && (item += p.page_items, true));
  }
}

template <class T, bool FP8, int D>
static hipError_t launch_append_t(const PagedAppendParams& pin, hipStream_t st) {
  PagedAppendParams p = pin;
  const PagedCache& c = p.c;
  p.row_groups = (p.q ? cdiv(c.Hq, kRowHeads) : 0) + (FP8 ? 0 : 2 * cdiv(c.Hkv, kRowHeads));
  // threads: a page's new rows in kAppendHold units each, or a wave's worth of units
  const int rows = c.n < c.page_size ? c.n : c.page_size;
  int nt = FP8 ? (rows * (D / 16) + 64 * kAppendHold - 1) / (64 * kAppendHold) * 64 : 256;
  nt = nt > kAppendThreads ? kAppendThreads : nt < 64 ? 64 : nt;
  const int64_t pages = FP8 ? (int64_t)p.page_items * 2 * c.Hkv : 0;
  const int64_t items = (int64_t)c.total * p.row_groups * (D / 16);
  const int64_t blocks = pages + (items + nt - 1) / nt;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL((paged_append_kernel<T, FP8, D>), dim3((unsigned)blocks), dim3(nt), 0, st, p, (int)pages);
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
// Attention, few columns: split over the rows
// ---------------------------------------------------------------------------
// A column is one (token, query head) of a KV head: column c of a sequence is token c / G and
// head c % G of the group of G heads.  The rows of all sequences, in units, are cut into `parts`
// equal runs (see Runs); one workgroup takes one run for NC tiles of 16 columns and one, two or
// four KV heads, and its waves share the heads and then the rows: each takes 32-row steps in
// turn, as two slices of 16 rows (a slice lies in one page), with no barrier until the merge
// at the end of a sequence or of the run.
// Equal runs: with fixed chunks of each sequence, 32 sequences of 1k to 32k rows left a tail of
// half-empty rounds, and grids sized for the page table's capacity were mostly empty.
// Several heads: rows of 128 bytes, one head's of many, reach 5.3 TB/s, four heads' side by side
// 6.0 (32 sequences of 16384 rows, 8 KV heads).
// * S^T = K Q^T on 16x16x32 MFMA, M = 16 rows, N = 16 columns: every K and V byte is read once
//   for all columns of the tile.
// * K rows go straight to registers in MFMA order, two steps ahead; e4m3 codes become 16-bit
//   values there (exact in both types).  V rows go through a wave-private LDS ring by direct
//   copies and come back transposed (ds_read_b64_tr_b16 / _tr_b8) as the operand of
//   O^T = V^T P^T.
// * A page's key scale multiplies its scores.  Its value scale multiplies P relative to the
//   largest seen so far, which O is kept in units of, so P stays in [0, 1] and no 16-bit value
//   leaves its type's range whatever the scales are.
// Bound by reading the cache (32 sequences of 1k to 32k rows, 32/8 heads of 128, 8 bits: 177 us,
// 6.2 TB/s; 16 bits 335 us, 6.6 TB/s); calls of some ten MB by the chain of dependent loads
// (lengths, page table, rows: 5 to 7 us) at the start and the merge at the end.

// Waves of a workgroup of the split kernel: eight where their rings fit the LDS.
__host__ __device__ constexpr int paged_waves(int d, bool fp8) { return d <= 128 || fp8 ? 8 : 4; }

template <int N>
__device__ __forceinline__ void wait_vmcnt_n() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Combine with the lanes 16 and 32 apart.
__device__ __forceinline__ float quarters_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_max(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

// log2-domain LSE of a sum of weights relative to m: -infinity if no row was seen, NaN if one of
// the scores was.
__device__ __forceinline__ float lse_of(float m, float sum) { return sum == 0.f ? -INFINITY : m + fast_log2(sum); }
// In a partial result infinity stands for NaN, which a maximum would pass over.
__device__ __forceinline__ float partial_lse(float lse2) { return lse2 != lse2 ? INFINITY : lse2; }

// Eight e4m3 codes as 16-bit values (exact)
template <class T>
__device__ __forceinline__ vec8<T> e4m3_to_16(uint32_t lo, uint32_t hi) {
  u32x4 r;
  if constexpr (std::is_same<T, half_t>::value) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  }
  return __builtin_bit_cast(vec8<T>, r);
}

typedef int i32x2 __attribute__((ext_vector_type(2)));

// Transposed LDS read of bytes: within 16 lanes, which read 8 rows x 16 columns (lane i row i / 2,
// columns 8 (i % 2) .. + 8), lane r gets column r, row j in byte j.
__device__ __forceinline__ u32x2 lds_tr8(const uint8_t* p) {
  typedef __attribute__((address_space(3))) i32x2 lds_i2;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)(p)));
}

__device__ __forceinline__ float lane_of(float x, int lane) { return __uint_as_float(lane_of(__float_as_uint(x), lane)); }

// Slice layout of V in LDS: 16 rows in 16-byte chunks, chunk index XOR-swizzled by the row so
// that a transposed read, whose half wave takes 8 rows of both slices, spreads over all banks.
template <bool FP8, int D>
struct VSlice {
  static constexpr int RB = FP8 ? D : 2 * D;                 // bytes of a row
  static constexpr int CPR = RB / 16;
  static constexpr int LOADS = (16 * CPR + 63) / 64;         // direct copies of 64 chunks
  static constexpr int BYTES = LOADS * 1024;                 // (a last half-used copy pads)
  __device__ static int swz(int row, int slice) {
    if (D == 96) return FP8 ? 0 : row & 3;
    if (!FP8) return row & (CPR < 16 ? CPR - 1 : 15);
    constexpr int RPL = CPR < 16 ? 16 / CPR : 1;             // rows per 256 bytes
    return (row / RPL + slice * (8 / RPL)) & (CPR - 1);
  }
};

// A pair of K pieces loaded by lines -> MFMA order.  Loaded: a = (lane n < 8 of a row of 16
// lanes: row n piece 0; n >= 8: row n - 8 piece 1), b = the same of rows 8 .. 15.  Wanted:
// a = row n piece 0, b = row n piece 1.  Lanes 8-15 of a take b from 8 lanes below, lanes 0-7 of
// b take a from 8 lanes above (row_ror:8).
__device__ __forceinline__ void unswap_lines(u32x4& a, u32x4& b) {
  u32x4 na, nb;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    na[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)a[i], (int)b[i], 0x128, 0xf, 0xc, false);
    nb[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)b[i], (int)a[i], 0x128, 0xf, 0x3, false);
  }
  a = na, b = nb;
}

// The units of all sequences, in order, cut into `parts` runs whose lengths differ by one at
// most: the first `extra` have `each` + 1.  Sequence b's units that lie in run g make up piece
// g + b: along the order either g or b grows by one, so pieces are numbered without gaps.
struct Runs {
  int64_t each, extra;
  __device__ Runs(int64_t units, int parts) {
    if (units >> 31) each = units / parts;
    else each = (uint32_t)units / (uint32_t)parts;
    extra = units - each * parts;
  }
  __device__ int64_t begin(int g) const { return g * each + (g < extra ? g : extra); }
  __device__ int of(int64_t unit) const {   // the run that a unit lies in
    const int64_t head = extra * (each + 1);
    if (unit < head) return (int)((unit >> 31) ? unit / (each + 1) : (uint32_t)unit / (uint32_t)(each + 1));
    return (int)(extra + ((unit - head) >> 31 ? (unit - head) / each : (uint32_t)(unit - head) / (uint32_t)each));
  }
};

__device__ __forceinline__ int cache_rows(const PagedCache& c, int b) { return min(max(c.seqlens[b], 0), c.capacity); }

// Packed sequences that both kernels share: the split kernel takes those of up to c.most tokens,
// the tile kernel the others.  Rows of sequence b for the split kernel:
__device__ __forceinline__ int split_rows(const PagedCache& c, int b) {
  int off, len = 0;
  if (c.most) seg_bounds(c.cu, b, c.total, off, len);
  return c.most && len > c.most ? 0 : cache_rows(c, b);
}

// Units of the sequences, by blocks of 64, one sequence per lane.  The first unit of a sequence has no
// rows: it stands for what starting and ending one costs (page table, scales, first rows, merge),
// so that runs that cross into the next sequence get fewer rows and all end together (24
// sequences of 77 to 4099 rows in 21 runs per head: 37.3 -> 35.3 us).
struct UnitBlocks {
  int unit[kBlocks], sum[kBlocks];   // a lane's units, and the inclusive sums within its block
  __device__ UnitBlocks(const PagedCache& c, int base, int unit_rows, int lane) {
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      const int b = base + 64 * k + lane;
      const int rows = b < c.B ? split_rows(c, b) : 0;
      unit[k] = rows > 0 ? cdiv(rows, unit_rows) + 1 : 0;
    }
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) sum[k] = base + 64 * k < c.B ? lanes_scan(unit[k]) : 0;
  }
  __device__ int total(int k) const { return (int)lane_of((uint32_t)sum[k], 63); }
  __device__ int before(int k, int at) const { return (int)(lane_of((uint32_t)sum[k], at) - lane_of((uint32_t)unit[k], at)); }
};

// Rows r0 .. r1 of the attention of one token i and query head h of sequence b, by one wave, row
// after row: the sums o of weights relative to m times values (element lane + 64 j in o[j]), and
// the weights' sum l.  For what the matrix kernels leave out: tokens past the stated longest
// sequence, and columns whose result is not finite under a causal mask, since in a matrix product
// a value that is not finite makes the columns that do not see its row NaN too (0 * infinity).
template <class T, bool FP8, int D>
__device__ void attend_alone(const PagedAttnParams& p, int b, int i, int h, int r0, int r1, float (&o)[(D + 63) / 64],
                             float& m, float& l) {
  const PagedCache& c = p.c;
  constexpr int DJ = (D + 63) / 64, CB = FP8 ? 1 : 2;
  const int lane = threadIdx.x & 63, hk = h / (c.Hq / c.Hkv);
  auto elem = [&](const char* row, int e) {
    if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)row)[e], 0);
    else return (float)((const T*)row)[e];
  };
  int off, len;
  token_range(c, b, off, len);
  const T* qrow = (const T*)p.q + (c.cu ? (int64_t)(off + i) * p.q_ss : b * p.q_sb + i * p.q_ss) + h * p.q_sh;
  float q[DJ];
#pragma unroll
  for (int j = 0; j < DJ; ++j) {
    const int e = lane + 64 * j;
    q[j] = e < D ? (float)qrow[e] * (p.negate_q ? -p.scale_log2 : p.scale_log2) : 0.f;
    o[j] = 0.f;
  }
  const int L = cache_rows(c, b), end = min(p.causal ? L - len + i + 1 : L, r1);
  m = -INFINITY, l = 0.f;
  for (int r = r0; r < end; ++r) {
    const int pid = c.table[b * c.table_sb + r / c.page_size], slot = r % c.page_size;
    if (pid < 0 || pid >= c.num_pages) continue;
    const char* k = (const char*)c.k + (pid * c.k_sp + hk * c.k_sh + slot * c.k_ss) * CB;
    const char* v = (const char*)c.v + (pid * c.v_sp + hk * c.v_sh + slot * c.v_ss) * CB;
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < DJ; ++j)
      if (lane + 64 * j < D) x = fmaf(q[j], elem(k, lane + 64 * j), x);
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
      if (lane + 64 * j < D) o[j] = fmaf(ev, elem(v, lane + 64 * j), o[j] * a);
  }
}

// NaN if one of the values is not finite, else 0
template <int N, class Acc>
__device__ __forceinline__ float not_finite(const Acc (&x)[N]) {
  float bad = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Acc) / sizeof(float)); ++i) bad = fmaf(x[k][i], 0.f, bad);
  return bad;
}

// ONE: one token per sequence, which sees every row (sequences with more are the combine kernel's).
template <class T, bool FP8, int D, int NC, bool ONE>
__global__ void __launch_bounds__(paged_waves(D, FP8) * 64, paged_waves(D, FP8) / 4)
paged_split_kernel(PagedAttnParams p) {
  constexpr int NW = paged_waves(D, FP8);
  constexpr int KS = D / 32;                     // 32-wide k-steps over the head dim
  constexpr int DBN = D / 16;
  using VS = VSlice<FP8, D>;
  // K registers of a slice: 16-byte pieces that cover 64 bytes of each of its 16 rows
  constexpr int KL = FP8 ? D / 64 : D / 32, KTAIL = FP8 ? (D % 64) / 32 : 0;   // (tail: 32 bytes of each row)
  constexpr bool LINE = KL >= 2;                 // pairs of pieces loaded as whole 128-byte lines
  constexpr int LPS = 2 * (KL + KTAIL + VS::LOADS);
  using V8 = vec8<T>;
  __shared__ __attribute__((aligned(1024))) uint8_t vsm[NW][4 * VS::BYTES];   // 2 steps x 2 slices
  __shared__ float m_s[NW][16], l_s[NW][16], inv_s[NW][16];
  static_assert(sizeof(vsm[0]) >= 16 * D * sizeof(float), "a wave's ring holds its partial O");

  const PagedCache& c = p.c;
  const int G = c.Hq / c.Hkv;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = tid >> 6;
  const int ws = __builtin_amdgcn_readfirstlane(w);
  const int l16 = lane & 15;
  const int g4 = lane >> 4;
  int rest = blockIdx.x;
  const int ct = rest % p.col_tiles;
  rest /= p.col_tiles;
  const int WH = p.wave_heads, NR = NW / WH;     // KV heads of the workgroup, waves on each
  const int hgroup = rest % (c.Hkv / WH);
  const int run = rest / (c.Hkv / WH);
  const int hkv = hgroup * WH + ws % WH;
  const int wr = ws / WH;

  // this run's first sequence and unit
  int b = 0, local = 0, left;
  if (p.direct) {        // one run is one sequence
    b = run, left = 0x7fffffff;
  } else {
    int64_t units = 0;
    for (int base = 0; base < c.B; base += 64 * kBlocks) {
      const UnitBlocks x(c, base, p.unit_rows, lane);
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) units += x.total(k);
    }
    const Runs runs(units, p.parts);
    const int64_t u0 = runs.begin(run);
    left = __builtin_amdgcn_readfirstlane((int)(runs.begin(run + 1) - u0));
    if (left <= 0) return;
    int64_t before = 0;
    bool found = false;
    for (int base = 0; base < c.B && !found; base += 64 * kBlocks) {
      const UnitBlocks x(c, base, p.unit_rows, lane);
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const auto past = __ballot(before + x.sum[k] > u0);
        if (!found && past) {
          const int at = __builtin_ctzll(past);
          b = base + 64 * k + at;
          local = (int)(u0 - before) - x.before(k, at);
          found = true;
        }
        before += x.total(k);
      }
    }
    b = __builtin_amdgcn_readfirstlane(b);
    local = __builtin_amdgcn_readfirstlane(local);
  }

  constexpr int CB = FP8 ? 1 : 2;
  const int k_ss = (int)c.k_ss * CB, v_ss = (int)c.v_ss * CB;   // row strides in bytes (below 2^23)
  const char* const kbase = (const char*)c.k + hkv * c.k_sh * CB;
  const char* const vbase = (const char*)c.v + hkv * c.v_sh * CB;
  const uint32_t k_page = (uint32_t)(c.k_sp * CB >> 4), v_page = (uint32_t)(c.v_sp * CB >> 4);   // 16-byte units
  const float* const kscale = FP8 ? c.k_scale + hkv * c.ks_sh : nullptr;
  const float* const vscale = FP8 ? c.v_scale + hkv * c.vs_sh : nullptr;
  // K: 16 bytes g4 of row l16 in piece t, or, by lines, of row l16 % 8 (+ 8 in the second of a
  // pair) and piece t + l16 / 8 (kline order; see unswap)
  const int kv0 = l16 * k_ss + g4 * 16;
  const int kvl = (l16 & 7) * k_ss + (g4 + 4 * (l16 >> 3)) * 16;
  int vv[2][VS::LOADS];   // byte of the chunk that each copy brings to this lane's place in a slice
#pragma unroll
  for (int I = 0; I < VS::LOADS; ++I) {
    const int q = I * 64 + lane, r = q / VS::CPR;
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)   // (past the slice's 16 rows: outside the resource, nothing is read)
      vv[sl][I] = r < 16 ? r * v_ss + ((q % VS::CPR) ^ VS::swz(r, sl)) * 16 : 0x7ffffff0;
  }
  uint8_t* const ring = &vsm[ws][0];

  u32x4 kreg[2][2][KL > 0 ? KL : 1];
  u32x2 ktail[2][2];
  // transposed V reads
  constexpr int VROW = VS::RB;
  const int kk = l16 >> 1;                                   // e4m3: row kk of the 8, slice kk / 4
  const int vr = FP8 ? 4 * g4 + (kk & 3) : 4 * g4 + (l16 >> 2);
  const uint8_t* vread = FP8 ? ring + (kk >> 2) * VS::BYTES + vr * VROW + 8 * (l16 & 1) : ring + vr * VROW + 8 * (l16 & 1);
  const int vc0 = FP8 ? VS::swz(vr, kk >> 2) : ((l16 >> 1) & 1) ^ VS::swz(vr, 0);

  for (; left > 0 && b < c.B; ++b, local = 0) {
    const int L = split_rows(c, b);
    const int take = min(left, (L > 0 ? cdiv(L, p.unit_rows) + 1 : 0) - local);
    left = p.direct ? 0 : left - take;
    const int row0 = max(local - 1, 0) * p.unit_rows, row1 = min(L, (local + take - 1) * p.unit_rows);
    int off, len;
    token_range(c, b, off, len);
    const int ncols = min(len, c.n) * G;
    if ((row0 >= row1 && !p.direct) || ct * NC * 16 >= ncols) continue;

    // rows below this one are seen by every column
    const int lim_first = !ONE && p.causal ? L - len + ct * NC * 16 / G + 1 : L;
    // queries of the columns as the B operand (n = column, k = head dim in K's order)
    V8 qreg[NC][KS];
    int lim[NC];         // rows below this one are seen by the column
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      const int col = (ct * NC + nc) * 16 + l16;
      const int i = col / G, h = hkv * G + col % G;
      const T* qrow = (const T*)p.q + (c.cu ? (int64_t)(off + i) * p.q_ss : b * p.q_sb + i * p.q_ss) + h * p.q_sh;
      lim[nc] = !ONE && p.causal ? L - len + i + 1 : L;
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const int e = FP8 && t < 2 * KL ? (t >> 1) * 64 + g4 * 16 + (t & 1) * 8 : t * 32 + g4 * 8;
        qreg[nc][t] = col < ncols ? ld8(qrow + e) : zero8<T>();
        if (p.negate_q) qreg[nc][t] = -qreg[nc][t];
      }
    }
    f32x4 oacc[NC][DBN];
    float m_run[NC], l_run[NC];
    float ref = 0.f;     // value scale that O is in units of
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      m_run[nc] = -INFINITY, l_run[nc] = 0.f;
#pragma unroll
      for (int i = 0; i < DBN; ++i) oacc[nc][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // Blocks of rows whose slices fit a wave's lanes, one per lane: slice i is half i % 2 of step
    // wr + NR * (i / 2).  Byte offsets of its first rows, the rows it has (0: none, or a page
    // outside the pool) and its scales.
    for (int k_begin = row0; k_begin < row1; k_begin += 1024 * NR) {
      const int k_end = min(row1, k_begin + 1024 * NR);
      const int nsteps = cdiv(k_end - k_begin, 32);
      int64_t koff = 0, voff = 0;
      int nrow = 0;
      float ksc = 1.f, vsc = 1.f;
      {
        const int r = k_begin + (wr + NR * (lane >> 1)) * 32 + (lane & 1) * 16;
        if (r < k_end) {
          const int page = r / c.page_size, slot = r - page * c.page_size;
          const int pid = c.table[b * c.table_sb + page];
          if (pid >= 0 && pid < c.num_pages) {
            nrow = min(16, k_end - r);
            koff = ((uint64_t)(uint32_t)pid * k_page << 4) + (uint32_t)(slot * k_ss);
            voff = ((uint64_t)(uint32_t)pid * v_page << 4) + (uint32_t)(slot * v_ss);
            if (FP8) {
              ksc = kscale[(uint64_t)(uint32_t)pid * (uint32_t)c.ks_sp];
              vsc = vscale[(uint64_t)(uint32_t)pid * (uint32_t)c.vs_sp];
            }
          }
        }
      }
      auto issue = [&](int jj, int buf) {   // the wave's step jj
#pragma unroll
        for (int sl = 0; sl < 2; ++sl) {
          const int i = 2 * jj + sl;
          const int n = (int)lane_of((uint32_t)nrow, i);
          const int64_t ko = (int64_t)(((uint64_t)lane_of((uint32_t)(koff >> 32), i) << 32) | lane_of((uint32_t)koff, i));
          const int64_t vo = (int64_t)(((uint64_t)lane_of((uint32_t)(voff >> 32), i) << 32) | lane_of((uint32_t)voff, i));
          const auto krs = make_rsrc(kbase + ko, n > 0 ? (uint32_t)((n - 1) * k_ss + D * CB) : 0);
          const auto vrs = make_rsrc(vbase + vo, n > 0 ? (uint32_t)((n - 1) * v_ss + D * CB) : 0);
#pragma unroll
          for (int t = 0; t < KL; ++t) {
            const bool pair = LINE && (t | 1) < KL;
            // whole lines are read once and evicted first; halves stay until the other half is read
            kreg[buf][sl][t] = pair ? __builtin_amdgcn_raw_buffer_load_b128(krs, kvl + (t & 1) * 8 * k_ss + (t & ~1) * 64, 0, 2)
                                    : __builtin_amdgcn_raw_buffer_load_b128(krs, kv0 + t * 64, 0, 0);
          }
          if constexpr (KTAIL)
            ktail[buf][sl] = __builtin_amdgcn_raw_buffer_load_b64(krs, l16 * k_ss + KL * 64 + g4 * 8, 0, 0);
#pragma unroll
          for (int I = 0; I < VS::LOADS; ++I)
            buffer_to_lds16<2>(vrs, vv[sl][I], ring + (buf * 2 + sl) * VS::BYTES + I * 1024);
        }
      };
      int j = wr;          // this wave's steps: wr, wr + NR, ...
      if (j < nsteps) issue(0, 0);
      if (j + NR < nsteps) issue(1, 1);
      auto step = [&](auto bufc, int jj) {
        constexpr int buf = decltype(bufc)::value;
        if (j + NR < nsteps) wait_vmcnt_n<LPS>();
        else wait_vmcnt_n<0>();
        f32x4 s[NC][2];
        float vfac[2], back = 1.f;
#pragma unroll
        for (int sl = 0; sl < 2; ++sl) {
          V8 kop[KS];
          if constexpr (LINE) {
#pragma unroll
            for (int t = 0; t + 1 < KL; t += 2) unswap_lines(kreg[buf][sl][t], kreg[buf][sl][t + 1]);
          }
          if constexpr (FP8) {
#pragma unroll
            for (int t = 0; t < KL; ++t) {
              kop[2 * t] = e4m3_to_16<T>(kreg[buf][sl][t][0], kreg[buf][sl][t][1]);
              kop[2 * t + 1] = e4m3_to_16<T>(kreg[buf][sl][t][2], kreg[buf][sl][t][3]);
            }
            if constexpr (KTAIL) kop[KS - 1] = e4m3_to_16<T>(ktail[buf][sl][0], ktail[buf][sl][1]);
          } else {
#pragma unroll
            for (int t = 0; t < KS; ++t) kop[t] = __builtin_bit_cast(V8, kreg[buf][sl][t]);
          }
#pragma unroll
          for (int nc = 0; nc < NC; ++nc) {
            s[nc][sl] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < KS; ++t) s[nc][sl] = mfma16(kop[t], qreg[nc][t], s[nc][sl]);
          }
        }
        const int n0 = (int)lane_of((uint32_t)nrow, 2 * jj), n1 = (int)lane_of((uint32_t)nrow, 2 * jj + 1);
        // scores stay unscaled until their exponent: max and mask commute with a positive factor
        float kfac[2] = {p.scale_log2, p.scale_log2};
        if constexpr (FP8) {
          kfac[0] = fmaxf(kfac[0] * lane_of(ksc, 2 * jj), 0x1p-126f), kfac[1] = fmaxf(kfac[1] * lane_of(ksc, 2 * jj + 1), 0x1p-126f);
          const float v0 = n0 > 0 ? lane_of(vsc, 2 * jj) : 0.f, v1 = n1 > 0 ? lane_of(vsc, 2 * jj + 1) : 0.f;
          const float now = fmaxf(ref, fmaxf(v0, v1));
          const float inv = now >= 0x1p-126f ? __builtin_amdgcn_rcpf(now) : 0.f;
          vfac[0] = v0 * inv, vfac[1] = v1 * inv, back = ref * inv;
          ref = now;
        }
        const int r0 = k_begin + j * 32;
        const bool whole = n0 == 16 && n1 == 16 && (ONE || r0 + 32 <= lim_first);   // every row seen by every column
        V8 pb[NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          if (!whole) {
#pragma unroll
            for (int sl = 0; sl < 2; ++sl)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = 4 * g4 + i;
                if (r >= (sl ? n1 : n0) || (!ONE && r0 + sl * 16 + r >= lim[nc])) s[nc][sl][i] = -INFINITY;
              }
          }
          float mx = fmaxf(fmaxf(fmaxf(s[nc][0][0], s[nc][0][1]), fmaxf(s[nc][0][2], s[nc][0][3])) * kfac[0],
                           fmaxf(fmaxf(s[nc][1][0], s[nc][1][1]), fmaxf(s[nc][1][2], s[nc][1][3])) * kfac[1]);
          mx = quarters_max(mx);
          const float m_new = fmaxf(m_run[nc], mx);
          const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
          float l = 0.f;
#pragma unroll
          for (int sl = 0; sl < 2; ++sl)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = fast_exp2(fmaf(s[nc][sl][i], kfac[sl], -m_use));
              l += e;
              pb[nc][sl * 4 + i] = (T)(FP8 ? e * vfac[sl] : e);
            }
          if (__any(m_new != m_run[nc]) || (FP8 && back != 1.f)) {
            const float alpha = fast_exp2(m_run[nc] - m_use);
            l_run[nc] *= alpha;
            m_run[nc] = m_new;
            const float f = FP8 ? alpha * back : alpha;
#pragma unroll
            for (int db = 0; db < DBN; ++db) oacc[nc][db] *= f;
          }
          l_run[nc] += l;
        }
        // O^T += V^T P^T over the 32 rows
#pragma unroll
        for (int db = 0; db < DBN; ++db) {
          V8 vop;
          if constexpr (FP8) {
            const u32x2 x = lds_tr8(vread + buf * 2 * VS::BYTES + ((db ^ vc0) << 4));
            vop = e4m3_to_16<T>(x[0], x[1]);
          } else {
            const T* v0 = (const T*)(vread + buf * 2 * VS::BYTES + ((vc0 ^ (2 * db)) << 4));
            vop = join8(lds_tr(v0), lds_tr((const T*)((const uint8_t*)v0 + VS::BYTES)));
          }
#pragma unroll
          for (int nc = 0; nc < NC; ++nc) oacc[nc][db] = mfma16(vop, pb[nc], oacc[nc][db]);
        }
        // LDS reads of this buffer must finish before the next copies overwrite it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (j + 2 * NR < nsteps) issue(jj + 2, buf);
        j += NR;
      };
      // two steps per trip so that the ring index is a compile-time constant
      for (int jj = 0; j < nsteps; jj += 2) {
        step(std::integral_constant<int, 0>{}, jj);
        if (j >= nsteps) break;
        step(std::integral_constant<int, 1>{}, jj + 1);
      }
    }

    // ---- the piece's partial output, normalised, and its log2-domain LSE; or the result ----
    const int64_t piece = (int64_t)(run + b) * c.Hkv;
    auto put = [&](int col, int kv, int d, f32x4 x) {
      if (!p.direct) {
        *reinterpret_cast<f32x4*>(p.part_o + ((piece + kv) * p.cols + col) * D + d) = x;
        return;
      }
      const vec4<T> y = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
      *reinterpret_cast<vec4<T>*>((T*)p.o + b * p.o_sb + col / G * p.o_ss + (kv * G + col % G) * p.o_sh + d) = y;
    };
    auto put_lse = [&](int col, int kv, float lse2) {
      if (!p.direct) p.part_m[(piece + kv) * p.cols + col] = partial_lse(lse2);
      else if (p.lse) p.lse[((int64_t)b * c.n + col / G) * c.Hq + kv * G + col % G] = lse2 * kLn2;
    };
    const bool masked = !ONE && p.causal && len > 1;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      const int col0 = (ct * NC + nc) * 16;
      const int nh = min(16, ncols - col0);
      // (NaN marks a column whose result is not finite, which the combine kernel takes on)
      const float l_tot = quarters_sum(masked ? l_run[nc] + not_finite(oacc[nc]) : l_run[nc]);
      if (NR == 1) {   // a wave has all of its head's rows
        const float f = l_tot == 0.f ? 0.f : (FP8 ? ref : 1.f) / l_tot;
        if (l16 < nh) {
#pragma unroll
          for (int db = 0; db < DBN; ++db) put(col0 + l16, hkv, db * 16 + 4 * g4, oacc[nc][db] * f);
          if (g4 == 0) put_lse(col0 + l16, hkv, lse_of(m_run[nc], l_tot));
        }
        continue;
      }
      // the waves of each head, added in their order; 16-byte chunks XOR-swizzled by the column
      if (lane < 16) {
        m_s[w][l16] = m_run[nc];
        l_s[w][l16] = l_tot;
      }
      __syncthreads();
      float M = -INFINITY, mw[NW], lw[NW];   // (of all waves: the reads then go out together)
#pragma unroll
      for (int i = 0; i < NW; ++i) mw[i] = m_s[i][l16], lw[i] = l_s[i][l16];
#pragma unroll
      for (int i = 0; i < NW; ++i) M = i % WH == ws % WH ? fmaxf(M, mw[i]) : M;
      const float M_use = (M == -INFINITY) ? 0.f : M;
      const float wscale = fast_exp2(m_run[nc] - M_use) * (FP8 ? ref : 1.f);
      constexpr int SW = D / 4 >= 16 && D != 96 ? 15 : 7;
      f32x4* part = reinterpret_cast<f32x4*>(ring);   // (the wave's ring is idle)
#pragma unroll
      for (int db = 0; db < DBN; ++db) part[l16 * (D / 4) + ((db * 4 + g4) ^ (l16 & SW))] = oacc[nc][db] * wscale;
      if (wr == 0 && lane < nh) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += i % WH == ws % WH ? lw[i] * fast_exp2(mw[i] - M_use) : 0.f;
        inv_s[w][l16] = sum == 0.f ? 0.f : 1.f / sum;
        put_lse(col0 + l16, hkv, lse_of(M_use, sum));
      }
      __syncthreads();
      for (int k = 0; k < WH; ++k) {
        for (int i = tid; i < nh * (D / 4); i += NW * 64) {
          const int n = i / (D / 4), q = i % (D / 4);
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int r = 0; r < NW; ++r)
            if (r < NR) o += reinterpret_cast<const f32x4*>(&vsm[k + r * WH][0])[n * (D / 4) + (q ^ (n & SW))];
          put(col0 + n, hgroup * WH + k, q * 4, o * inv_s[k][n]);
        }
      }
      __syncthreads();   // before the ring and the statistics are written again
    }
  }
}

// ---------------------------------------------------------------------------
// Attention, many columns: tiles of keys shared by a workgroup
// ---------------------------------------------------------------------------
// One workgroup takes 128 columns (see above) of one sequence and KV head, 32 to a wave (or 64, and
// two waves share a column's rows: half of the matrix units would idle otherwise), and
// walks tiles of 64 or 32 rows; with few workgroups, `splits` of them share a column tile's rows.
// * Each wave brings a slice of the tile (16 rows of one page, or half of one) from the cache: its
//   page and scales are scalars, its lanes' places in the page constants, and e4m3 codes become
//   16-bit values once, on the way to LDS, not once per wave that reads them.  Loads of a tile
//   run a whole tile ahead, its page number two.
// * S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMA; the S^T accumulators are P^T's operand in
//   place (fal_common.h).
// * The running maximum that exponents are taken from moves only when a score passes it by 8:
//   P reaches 2^8 at most, and the accumulators are rarely rescaled.
// * Scales as in the split kernel: the value factor enters the exponent, and each slice's sum is
//   divided by it again for l.
// * Each group of LDS reads goes out before the products of the group before it (chunk of 1024
//   tokens behind 8192 rows, 32/8 heads of 128, 8 bits: 234 -> 184 us).
// Bound by the vector units (ten instructions per matrix instruction, 32 % of the matrix units'
// time used at 234 us): that chunk runs at 790 TFLOP/s, in 16 bits at 860.
constexpr int kTileCols = 128;
// Tiles in LDS: swizzled rows, or for head dim 96 rows padded to 208 bytes, of which any sixteen
// start on different 16-byte pieces of the 256 that the banks hold.
template <int D>
struct PagedTile : SwizzledTile<D> {
  static constexpr int LD = D;
};
template <>
struct PagedTile<96> {
  static constexpr int LD = 104;
  __device__ static int offset(int r, int c) { return r * LD + c * 8; }
};
constexpr int tile_rows(int d) { return d > 128 ? 32 : 64; }   // (head dim 256: registers)

// The kernel's parameter block, read again where it is named: a path that is hardly ever taken
// then keeps nothing of it in registers all the way (a kernel's first argument opens the segment).
template <class P>
__device__ __forceinline__ const P& args_again() {
  auto a = (const __attribute__((address_space(4))) P*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const P*)a;
}

// Column `col` of sequence b and KV head hkv over the rows r0 .. r1 of a split, by one wave (see
// attend_alone).  Not inlined: it is hardly ever reached, and inlined it took registers from the
// loop (chunk of 1024 tokens behind 8192 rows 185 -> 193 us).
template <class T, bool FP8, int D>
__device__ __attribute__((noinline)) void column_again(const PagedAttnParams& p, int b, int hkv, int col, int split, int r0, int r1) {
  const PagedCache& c = p.c;
  const int G = c.Hq / c.Hkv, i = col / G, h = hkv * G + col % G, lane = threadIdx.x & 63;
  int off, len;
  token_range(c, b, off, len);
  float o[(D + 63) / 64], m, l;
  attend_alone<T, FP8, D>(p, b, i, h, r0, r1, o, m, l);
  const float inv = l == 0.f ? 0.f : 1.f / l, lse2 = lse_of(m, l);
  const int64_t row = ((c.cu ? off : (int64_t)b * c.n) + i) * c.Hq + h;
  T* orow = (T*)p.o + (c.cu ? (int64_t)(off + i) * p.o_ss : b * p.o_sb + i * p.o_ss) + h * p.o_sh;
#pragma unroll
  for (int j = 0; j < (D + 63) / 64; ++j) {
    const int d = lane + 64 * j;
    if (d >= D) continue;
    if (p.splits > 1) p.part_o[(row * p.splits + split) * D + d] = o[j] * inv;
    else orow[d] = (T)(o[j] * inv);
  }
  if (lane) return;
  if (p.splits > 1) p.part_m[row * p.splits + split] = partial_lse(lse2);
  else if (p.lse) p.lse[row] = lse2 * kLn2;
}

// Item `item` of the tiles of tc columns of packed tokens: sequence (its first token, tokens
// and rows too: all of its loads go out at once) and tile; false past the last.
// In the order of the tiles' numbers, the last first (they see the most rows), by 256 sequences.
// The tiles numbered x and more are the sum over the sequences of max(tiles - x, 0): the item's
// number is the largest x of which that sum passes it.  (A workgroup for every sequence and tile
// of the longest one's: 255 tokens and a prompt of 8192, 3065 us; by the tiles there are 948.
// Not inlined: inlined it cost the loop behind it (chunk of 1024 tokens 184 -> 191 us, so 186).)
struct TileItem {
  int b, ct, off, len, rows;   // b < 0: none
};
__device__ __attribute__((noinline)) TileItem tile_of_item(const PagedAttnParams& p, int tc, int64_t item) {
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 63, G = c.Hq / c.Hkv;
  for (int base = 0; base < c.B; base += 64 * kBlocks) {
    int n[kBlocks], first[kBlocks], tokens[kBlocks], rows[kBlocks], most = 0;
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      const int s = base + 64 * k + lane;
      first[k] = tokens[k] = rows[k] = 0;
      if (s < c.B) seg_bounds(c.cu, s, c.total, first[k], tokens[k]), rows[k] = cache_rows(c, s);
      n[k] = tokens[k] > c.most ? cdiv(tokens[k] * G, tc) : 0;
      most = max(most, n[k]);
    }
    auto from = [&](int x) {
      int sum = 0;
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) sum += max(n[k] - x, 0);
      return lane_of((uint32_t)lanes_scan(sum), 63);
    };
    const uint32_t all = from(0);
    if (item >= all) {
      item -= all;
      continue;
    }
    int bit = 0, x = 0;
    while (bit < 30 && __ballot(most >> bit)) ++bit;
    while (--bit >= 0)
      if (from(x | 1 << bit) > item) x |= 1 << bit;
    uint32_t r = (uint32_t)item - from(x + 1);
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      auto more = __ballot(n[k] > x);
      const uint32_t cnt = __builtin_popcountll(more);
      if (r < cnt) {
        for (; r; --r) more &= more - 1;
        const int at = __builtin_ctzll(more);
        return {base + 64 * k + at, x, (int)lane_of((uint32_t)first[k], at), (int)lane_of((uint32_t)tokens[k], at),
                (int)lane_of((uint32_t)rows[k], at)};
      }
      r -= cnt;
    }
    break;   // (offsets that are not monotone, whose tiles' sum passed 32 bits)
  }
  return {-1, 0, 0, 0, 0};
}

template <class T, bool FP8, int D, int RS>
__global__ void __launch_bounds__(256, D > 128 ? 1 : 2)
paged_tile_kernel(PagedAttnParams p) {
  constexpr int DB = D / 32, KS = D / 16;
  constexpr int RB = FP8 ? D : 2 * D, CPR = RB / 16;         // bytes of a cache row, its 16-byte pieces
  constexpr int TR = tile_rows(D), NS = TR / 16, NW = NS / RS;   // rows and slices of a tile, slices of a wave
  constexpr int RW = TR / 4;                                 // rows that a wave brings
  constexpr int LOADS = (RW * CPR + 63) / 64;                // pieces per lane of those
  constexpr int CB = FP8 ? 1 : 2;
  using V8 = vec8<T>;
  using Tile = PagedTile<D>;
  constexpr int TC = kTileCols / RS;                         // columns of a tile
  __shared__ __attribute__((aligned(1024))) T ksm[2][TR * Tile::LD], vsm[2][TR * Tile::LD];
  __shared__ float ssm[2][NS][2];                            // per slice: key and value scale (-1: no page)

  const PagedCache& c = p.c;
  const int G = c.Hq / c.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if ((int)blockIdx.x >= p.tile_blocks) {   // packed rows outside every sequence
    const int lo = min(max(c.cu[0], 0), c.total), hi = max(min(max(c.cu[c.B], 0), c.total), lo);
    for (int64_t r = ((int)blockIdx.x - p.tile_blocks) * 4 + w; r < (int64_t)(lo + c.total - hi) * c.Hq; r += 4 * p.rest_blocks) {
      const int64_t t = r / c.Hq < lo ? r / c.Hq : r / c.Hq - lo + hi;
      const int h = (int)(r % c.Hq);
      for (int d = lane; d < D; d += 64) ((T*)p.o + t * p.o_ss + h * p.o_sh)[d] = (T)0.f;
      if (p.lse && lane == 0) p.lse[t * c.Hq + h] = -INFINITY;
    }
    return;
  }
  int rest = blockIdx.x;
  const int hkv = rest % c.Hkv;
  rest /= c.Hkv;
  const int split = rest % p.splits;
  rest /= p.splits;
  const char* const kbase = (const char*)c.k + hkv * c.k_sh * CB;
  const char* const vbase = (const char*)c.v + hkv * c.v_sh * CB;
  const float* const kscale = FP8 ? c.k_scale + hkv * c.ks_sh : nullptr;
  const float* const vscale = FP8 ? c.v_scale + hkv * c.vs_sh : nullptr;
  const uint32_t k_page = (uint32_t)(c.k_sp * CB >> 4), v_page = (uint32_t)(c.v_sp * CB >> 4);   // 16-byte units
  const int step_pages = TR / c.page_size, step_rows = TR - step_pages * c.page_size;
  // column tiles, those that see the most rows first (packed tokens: more than one only where
  // sequences overlap or pass the stated longest)
  int64_t item = rest;
  do {
    TileItem it;
    if (c.cu) it = tile_of_item(args_again<PagedAttnParams>(), TC, item);
    else it = {rest % c.B, p.tile_cols - 1 - rest / c.B, 0, c.n, cache_rows(c, rest % c.B)};
    const int b = __builtin_amdgcn_readfirstlane(it.b), ct = __builtin_amdgcn_readfirstlane(it.ct);
    const int off = __builtin_amdgcn_readfirstlane(it.off), len = __builtin_amdgcn_readfirstlane(it.len);
    const int L = __builtin_amdgcn_readfirstlane(it.rows);
    if (b < 0) return;
    const int ncols = len * G;
    const int col_last = min(ncols, (ct + 1) * TC) - 1;
    const int k_hi = max(p.causal ? L - len + col_last / G + 1 : L, 0);
    const int tiles = cdiv(k_hi, TR);
    const int t0 = (int)((int64_t)tiles * split / p.splits), t1 = (int)((int64_t)tiles * (split + 1) / p.splits);

    // this wave's columns
    const int wc = w % (4 / RS), wx = w / (4 / RS) * NW;     // its 32 columns and its first slice
    const int col = ct * TC + wc * 32 + l32, i_tok = col / G, head = hkv * G + col % G;
    const bool have = col < ncols, active = ct * TC + wc * 32 < ncols;
    const int lim = p.causal ? L - len + i_tok + 1 : L;
    const int lim_first = p.causal ? L - len + (ct * TC + wc * 32) / G + 1 : L;
    V8 qreg[KS];
    const T* qrow = (const T*)p.q + (c.cu ? (int64_t)(off + i_tok) * p.q_ss : b * p.q_sb + i_tok * p.q_ss) + head * p.q_sh;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      qreg[t] = have ? ld8(qrow + t * 16 + hh * 8) : zero8<T>();
      if (p.negate_q) qreg[t] = -qreg[t];
    }
    f32x16 oacc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) oacc[i] = zero_f16();
    float m_ref = -INFINITY, l_run = 0.f, ref = 0.f;

    // staging: this lane's pieces of the wave's slice
    const int k_ss = (int)c.k_ss * CB, v_ss = (int)c.v_ss * CB;
    int kv[LOADS], vv[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int e = i * 64 + lane, r = e / CPR, u = e % CPR;
      kv[i] = r < RW ? r * k_ss + u * 16 : 0x7ffffff0;
      vv[i] = r < RW ? r * v_ss + u * 16 : 0x7ffffff0;
    }
    // the wave's slice of the tile whose page number is asked for next: its first row, and that
    // row's page and place in it
    int row = t0 * TR + w * RW, page = row / c.page_size, slot = row - page * c.page_size;
    struct Slice { int pid, slot, rows; };
    auto next_slice = [&]() {
      Slice x{-1, slot, 0};
      if (row < min(k_hi, t1 * TR)) {
        const int pid = c.table[b * c.table_sb + page];
        if (pid >= 0 && pid < c.num_pages) x.pid = pid, x.rows = min(RW, k_hi - row);
      }
      row += TR, page += step_pages, slot += step_rows;
      if (slot >= c.page_size) slot -= c.page_size, ++page;
      return x;
    };
    u32x4 kreg[LOADS], vreg[LOADS];
    float ksc, vsc;
    auto fetch = [&](Slice x) {
      const uint32_t pid = x.pid >= 0 ? x.pid : 0;
      const auto krs = make_rsrc(kbase + ((uint64_t)pid * k_page << 4) + (uint32_t)(x.slot * k_ss),
                                 x.rows > 0 ? (uint32_t)((x.rows - 1) * k_ss + RB) : 0);
      const auto vrs = make_rsrc(vbase + ((uint64_t)pid * v_page << 4) + (uint32_t)(x.slot * v_ss),
                                 x.rows > 0 ? (uint32_t)((x.rows - 1) * v_ss + RB) : 0);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        kreg[i] = __builtin_amdgcn_raw_buffer_load_b128(krs, kv[i], 0, 0);
        vreg[i] = __builtin_amdgcn_raw_buffer_load_b128(vrs, vv[i], 0, 0);
      }
      ksc = 1.f, vsc = x.rows > 0 ? 1.f : -1.f;
      if (FP8 && x.rows > 0) {
        ksc = kscale[(uint64_t)pid * (uint32_t)c.ks_sp];
        vsc = vscale[(uint64_t)pid * (uint32_t)c.vs_sp];
      }
    };
    auto stage = [&](int buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 64 + lane, r = e / CPR, u = e % CPR, row = w * RW + r;
        if (RW * CPR % 64 != 0 && r >= RW) continue;
        if constexpr (FP8) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            st_u4(&ksm[buf][Tile::offset(row, 2 * u + x)], __builtin_bit_cast(u32x4, e4m3_to_16<T>(kreg[i][2 * x], kreg[i][2 * x + 1])));
            st_u4(&vsm[buf][Tile::offset(row, 2 * u + x)], __builtin_bit_cast(u32x4, e4m3_to_16<T>(vreg[i][2 * x], vreg[i][2 * x + 1])));
          }
        } else {
          st_u4(&ksm[buf][Tile::offset(row, u)], kreg[i]);
          st_u4(&vsm[buf][Tile::offset(row, u)], vreg[i]);
        }
      }
      if (lane == 0 && w * RW % 16 == 0) ssm[buf][w * RW / 16][0] = ksc, ssm[buf][w * RW / 16][1] = vsc;
    };

    if (t0 < t1) {
      const Slice s0 = next_slice(), s1 = next_slice();
      Slice coming = next_slice();
      fetch(s0);
      stage(0);
      fetch(s1);
      __syncthreads();
      auto step = [&](auto bufc, int t) {
        constexpr int buf = decltype(bufc)::value;
        if (active) {
          // S^T: element i of block mb is row mb * 32 + (i / 4) * 8 + hh * 4 + i % 4, column l32
          constexpr int MB = TR / 32 / RS;
          const T* const kt = &ksm[buf][wx * 16 * Tile::LD];
          const T* const vt = &vsm[buf][wx * 16 * Tile::LD];
          f32x16 s[MB];
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) s[mb] = zero_f16();
          constexpr int KB = 2;   // k-steps whose operands are read together, one group ahead
          V8 ka[2][MB][KB];
          auto read_k = [&](int g) {
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
              for (int i = 0; i < KB; ++i)
                ka[g & 1][mb][i] = ld8(kt + Tile::offset(mb * 32 + l32, (g * KB + i) * 2 + hh));
          };
          read_k(0);
#pragma unroll
          for (int g = 0; g < KS / KB; ++g) {
            if (g + 1 < KS / KB) read_k(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < KB; ++i)
#pragma unroll
              for (int mb = 0; mb < MB; ++mb) s[mb] = mfma32(ka[g & 1][mb][i], qreg[g * KB + i], s[mb]);
          }
          // V operands of the first slice, read while the softmax runs
          constexpr int VG = DB < 4 ? DB : 4, VH = DB / VG;   // head-dim blocks read together, groups of them
          V8 va[2][VG];
          const int tr = hh * 4 + ((lane & 15) >> 2), tc = ((lane & 16) >> 3) + ((lane & 3) >> 1);
          auto read_v = [&](int g) {
            const int x = g / VH;
#pragma unroll
            for (int i = 0; i < VG; ++i) {
              const int ch = (g % VH * VG + i) * 4 + tc;
              va[g & 1][i] = join8(lds_tr(vt + Tile::offset(x * 16 + tr, ch) + (lane & 1) * 4),
                                   lds_tr(vt + Tile::offset(x * 16 + 8 + tr, ch) + (lane & 1) * 4));
            }
          };
          read_v(0);
          __builtin_amdgcn_sched_barrier(0);
          // the wave's slice x: elements 8 (x % 2) .. + 8 of block x / 2
          float kfac[NW], vlog[NW], vinv[NW], back = 1.f;
          bool whole = (t + 1) * TR <= lim_first;
          if constexpr (FP8) {
            float v[NW], now = ref;
#pragma unroll
            for (int x = 0; x < NW; ++x) {
              kfac[x] = fmaxf(p.scale_log2 * ssm[buf][wx + x][0], 0x1p-126f);
              v[x] = ssm[buf][wx + x][1];
              whole = whole && __builtin_amdgcn_readfirstlane(__float_as_int(v[x])) >= 0;
              now = fmaxf(now, v[x]);
            }
            const float inv = now >= 0x1p-126f ? __builtin_amdgcn_rcpf(now) : 0.f;
            back = ref * inv;
            ref = now;
#pragma unroll
            for (int x = 0; x < NW; ++x) {   // (a value scale 2^60 below the largest counts as that)
              const float f = fmaxf(v[x] * inv, 0x1p-60f);
              vlog[x] = fast_log2(f), vinv[x] = __builtin_amdgcn_rcpf(f);
            }
          } else {
#pragma unroll
            for (int x = 0; x < NW; ++x) {
              kfac[x] = p.scale_log2, vlog[x] = 0.f, vinv[x] = 1.f;
              whole = whole && __builtin_amdgcn_readfirstlane(__float_as_int(ssm[buf][wx + x][1])) >= 0;
            }
          }
          if (!whole) {
#pragma unroll
            for (int x = 0; x < NW; ++x) {
              const bool none = ssm[buf][wx + x][1] < 0.f;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = t * TR + (wx + x) * 16 + (i / 4) * 8 + hh * 4 + i % 4;
                if (none || r >= lim) s[x / 2][(x & 1) * 8 + i] = -INFINITY;
              }
            }
          }
          float mx = -INFINITY;
#pragma unroll
          for (int x = 0; x < NW; ++x) {
            const f32x16& y = s[x / 2];
            const int o = (x & 1) * 8;
            float a = y[o];
#pragma unroll
            for (int i = 1; i < 8; ++i) a = __builtin_elementwise_maximum(a, y[o + i]);
            mx = fmaxf(mx, a * kfac[x]);
          }
          mx = pair_max(mx);
          if (__any(mx > m_ref + 8.f) || (FP8 && back != 1.f)) {
            const float m_new = mx > m_ref ? mx : m_ref;
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_ref - m_new);
            m_ref = m_new;
            l_run *= alpha;
            const float f = alpha * back;
#pragma unroll
            for (int i = 0; i < DB; ++i) oacc[i] *= f;
          }
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
          V8 pb[NW];
#pragma unroll
          for (int x = 0; x < NW; ++x) {
            const float sub = FP8 ? vlog[x] - m_use : -m_use;
            float l = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float e = fast_exp2(fmaf(s[x / 2][(x & 1) * 8 + i], kfac[x], sub));
              l += e;
              pb[x][i] = (T)e;
            }
            l_run = FP8 ? fmaf(l, vinv[x], l_run) : l_run + l;
          }
          // O^T += V^T P^T
#pragma unroll
          for (int g = 0; g < NW * VH; ++g) {
            if (g + 1 < NW * VH) read_v(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < VG; ++i)
              oacc[g % VH * VG + i] = mfma32(va[g & 1][i], pb[g / VH], oacc[g % VH * VG + i]);
          }
        }
        if (t + 1 < t1) {
          stage(buf ^ 1);
          fetch(coming);
          coming = next_slice();
        }
        __syncthreads();
      };
      // two tiles per trip so that the buffer is a compile-time constant
      for (int t = t0; t < t1; t += 2) {
        step(std::integral_constant<int, 0>{}, t);
        if (t + 1 < t1) step(std::integral_constant<int, 1>{}, t + 1);
      }
    }

    const bool masked = p.causal && len > 1;
    // (NaN marks a column whose result is not finite)
    l_run = pair_sum(masked ? l_run + not_finite(oacc) : l_run);
    if constexpr (RS == 2) {   // the two waves of a column meet: the second one's sums go through LDS
      float* const mls = reinterpret_cast<float*>(&vsm[0][0]) + wc * 128;
      f32x4* const sums = reinterpret_cast<f32x4*>(&ksm[0][0]) + wc * (DB * 4 * 64);
      static_assert(sizeof(ksm) >= 2 * DB * 4 * 64 * sizeof(f32x4), "two waves' sums fit");
      if (wx) {
        mls[lane] = m_ref, mls[64 + lane] = l_run;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = FP8 ? ref : 1.f;
            sums[(db * 4 + i) * 64 + lane] =
                f32x4{oacc[db][4 * i], oacc[db][4 * i + 1], oacc[db][4 * i + 2], oacc[db][4 * i + 3]} * f;
          }
      }
      __syncthreads();
      if (!wx) {
        const float m2 = mls[lane], m = fmaxf(m_ref, m2), use = m == -INFINITY ? 0.f : m;
        const float a1 = fast_exp2(m_ref - use), a2 = fast_exp2(m2 - use);
        m_ref = m;
        l_run = l_run * a1 + mls[64 + lane] * a2;
        const float f = a1 * (FP8 ? ref : 1.f);
        ref = 1.f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) oacc[db][i] = oacc[db][i] * f + sums[(db * 4 + i / 4) * 64 + lane][i % 4] * a2;
      }
      __syncthreads();   // before the next columns' tiles are staged
    }
    auto marked = __ballot(masked && have && !wx && hh == 0 && l_run != l_run);
    const int64_t t_row = c.cu ? off : (int64_t)b * c.n;       // the sequence's first token
    if (have && !wx && !(marked >> l32 & 1)) {
      const float f = l_run == 0.f ? 0.f : (FP8 ? ref : 1.f) / l_run;
      const float lse2 = lse_of(m_ref, l_run);
      const int64_t row = (t_row + i_tok) * c.Hq + head;
      T* orow = (T*)p.o + (c.cu ? (int64_t)(off + i_tok) * p.o_ss : b * p.o_sb + i_tok * p.o_ss) + head * p.o_sh;
      float* part = p.part_o + (row * p.splits + split) * D;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = db * 32 + i * 8 + hh * 4;
          const f32x4 x = f32x4{oacc[db][4 * i], oacc[db][4 * i + 1], oacc[db][4 * i + 2], oacc[db][4 * i + 3]} * f;
          if (p.splits > 1) *reinterpret_cast<f32x4*>(part + d) = x;
          else *reinterpret_cast<vec4<T>*>(orow + d) = vec4<T>{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
        }
      if (hh == 0) {
        if (p.splits > 1) p.part_m[row * p.splits + split] = partial_lse(lse2);
        else if (p.lse) p.lse[row] = lse2 * kLn2;
      }
    }
    for (; marked; marked &= marked - 1)
      column_again<T, FP8, D>(args_again<PagedAttnParams>(), b, hkv, ct * TC + wc * 32 + __builtin_ctzll(marked), split, t0 * TR, t1 * TR);
  } while (c.cu && (item += p.items, true));
}

// Merge the pieces' partial outputs of (token, query head) rows, W waves to a row and four waves
// to a workgroup.  Each wave takes every W-th piece, eight of them in flight, with weights
// relative to its own largest LSE; four waves of a row meet in LDS in a fixed order.  (One wave
// for rows of few pieces: 10240 rows of about four, 34 -> 13 us.)
template <class T, bool FP8, int D, int W>
__global__ void __launch_bounds__(256)
paged_combine_kernel(PagedAttnParams p) {
  constexpr int DJ = (D + 63) / 64;
  constexpr int CH = 8;
  __shared__ float m_s[4], l_s[4], o_s[4][D];
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t row = (int64_t)blockIdx.x * (4 / W) + (W == 4 ? 0 : wave);
  if (row >= (c.most ? (int64_t)c.B * c.most : c.total) * c.Hq) return;
  const int w = W == 4 ? wave : 0;
  const int h = (int)(row % c.Hq);
  int t = (int)(row / c.Hq), b = 0, i = 0, ns = 0, off = 0, len = 1;
  bool in;
  if (c.most) {   // the sequences of few tokens, each with places for c.most
    b = t / c.most, i = t - b * c.most;
    token_range(c, b, off, len);
    if (i >= len || len > c.most) return;
    in = true, t = off + i, row = (int64_t)t * c.Hq + h;
  } else {
    in = token_place(c, t, b, i);
    if (in) token_range(c, b, off, len);
  }
  const bool alone = in && (i >= c.n || (c.n == 1 && len > 1));   // past the stated longest sequence
  const int G = c.Hq / c.Hkv;
  int64_t base = 0, step = (int64_t)c.Hkv * p.cols;
  if (in && !alone) {   // this sequence's pieces
    int64_t units = 0, first = 0;
    int mine = 0;
    for (int at = 0; at < c.B; at += 64 * kBlocks) {
      const UnitBlocks x(c, at, p.unit_rows, lane);
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const int l = b - at - 64 * k;
        if (l >= 0 && l < 64) {
          first = units + x.before(k, l);
          mine = (int)lane_of((uint32_t)x.unit[k], l);
        }
        units += x.total(k);
      }
    }
    if (mine > 0) {
      const Runs runs(units, p.parts);
      int g0 = runs.of(first);
      if (runs.begin(g0 + 1) == first + 1) ++g0;   // (nothing but the unit without rows)
      ns = runs.of(first + mine - 1) - g0 + 1;
      base = ((int64_t)(g0 + b) * c.Hkv + h / G) * p.cols + i * G + h % G;
    }
  }
  float acc[DJ];
#pragma unroll
  for (int j = 0; j < DJ; ++j) acc[j] = 0.f;
  float M = -INFINITY, wsum = 0.f;
  for (int s0 = w; s0 < ns; s0 += W * CH) {
    float pm[CH], x[CH][DJ];
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const bool ok = s0 + W * u < ns;
      const int64_t at = base + (s0 + W * u) * step;
      pm[u] = ok ? p.part_m[at] : -INFINITY;
#pragma unroll
      for (int j = 0; j < DJ; ++j) x[u][j] = (ok && lane + 64 * j < D) ? p.part_o[at * D + lane + 64 * j] : 0.f;
    }
    float cm = -INFINITY;
#pragma unroll
    for (int u = 0; u < CH; ++u) cm = fmaxf(cm, pm[u]);
    const float Mn = fmaxf(M, cm);
    if (Mn == -INFINITY) continue;
    const float r = fast_exp2(M - Mn);
    wsum *= r;
#pragma unroll
    for (int j = 0; j < DJ; ++j) acc[j] *= r;
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const float wgt = fast_exp2(pm[u] - Mn);
      wsum += wgt;
#pragma unroll
      for (int j = 0; j < DJ; ++j) acc[j] = fmaf(wgt, x[u][j], acc[j]);
    }
    M = Mn;
  }
  // a piece that is not finite (see attend_alone): every wave of the row sees the same
  bool again = false;
  if (p.causal && c.n > 1)
    for (int s0 = 0; s0 < ns; s0 += 64)
      again = again || __any(s0 + lane < ns && p.part_m[base + (s0 + lane) * step] == INFINITY);
  if (alone || again) {
    if (w == 0) attend_alone<T, FP8, D>(p, b, i, h, 0, 0x7fffffff, acc, M, wsum);
    else M = -INFINITY, wsum = 0.f;
    if (w)
#pragma unroll
      for (int j = 0; j < DJ; ++j) acc[j] = 0.f;
  }
  T* orow = (T*)p.o + (c.cu ? t * p.o_ss : b * p.o_sb + i * p.o_ss) + h * p.o_sh;
  if constexpr (W == 1) {
    const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
#pragma unroll
    for (int j = 0; j < DJ; ++j)
      if (lane + 64 * j < D) orow[lane + 64 * j] = (T)(acc[j] * inv);
    if (p.lse && lane == 0) p.lse[row] = lse_of(M, wsum) * kLn2;
  } else {
    if (lane == 0) m_s[w] = M, l_s[w] = wsum;
#pragma unroll
    for (int j = 0; j < DJ; ++j)
      if (lane + 64 * j < D) o_s[w][lane + 64 * j] = acc[j];
    __syncthreads();
    const float top = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
    float f[4], sum = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f[u] = m_s[u] == -INFINITY ? 0.f : fast_exp2(m_s[u] - top);
      sum += l_s[u] * f[u];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int d = threadIdx.x; d < D; d += 256)
      orow[d] = (T)((o_s[0][d] * f[0] + o_s[1][d] * f[1] + o_s[2][d] * f[2] + o_s[3][d] * f[3]) * inv);
    if (p.lse && threadIdx.x == 0) p.lse[row] = lse_of(top, sum) * kLn2;
  }
}

// Merge the tile kernel's splits, four elements of one (token, query head) per thread.
template <class T, int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(PagedAttnParams p) {
  const PagedCache& c = p.c;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (D / 4);
  const int d = (int)(i % (D / 4)) * 4;
  if (row >= (int64_t)c.total * c.Hq) return;
  const int t = (int)(row / c.Hq), h = (int)(row % c.Hq);
  int b, n;
  const bool in = token_place(c, t, b, n);
  if (in && c.most) {   // the split kernel's
    int off, len;
    token_range(c, b, off, len);
    if (len <= c.most) return;
  }
  const float* pm = p.part_m + row * p.splits;
  const f32x4* po = reinterpret_cast<const f32x4*>(p.part_o + row * p.splits * D + d);
  float M = -INFINITY, sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, pm[s]);
    if (M > -INFINITY)
      for (int s = 0; s < p.splits; ++s) {
        const float w = fast_exp2(pm[s] - M);
        sum += w;
        o += po[s * (D / 4)] * w;
      }
  }
  o *= sum == 0.f ? 0.f : 1.f / sum;
  T* orow = (T*)p.o + (c.cu ? t * p.o_ss : b * p.o_sb + n * p.o_ss) + h * p.o_sh;
  *reinterpret_cast<vec4<T>*>(orow + d) = vec4<T>{(T)o[0], (T)o[1], (T)o[2], (T)o[3]};
  if (p.lse && d == 0) p.lse[row] = lse_of(M, sum) * kLn2;
}

constexpr int kSplitCols = 32;      // most columns of a KV head that the split kernel takes
constexpr int kDirectRows = 2048;   // longest caches that one workgroup takes whole

PagedPlan paged_plan(int64_t B, int64_t seqlen, int64_t total, int64_t Hq, int64_t Hkv, int64_t capacity, int d, bool fp8,
                     bool packed, int ncu) {
  PagedPlan r{};
  const int64_t G = Hq / Hkv;
  int64_t cols = (seqlen > 0 ? seqlen : 1) * G;
  if (cols > kSplitCols) {
    // Sequences of few tokens (one tile of 16 columns, or one token) among packed longer ones go
    // to the split kernel, as a prompt's chunk and running sequences make up one step: where all
    // but the longest have that few on average (255 tokens behind 2000 rows and 2048 of a prompt
    // 403 -> 296 us; 63 behind 8000 364 -> 250).  Elsewhere the second pair of launches finds little to do.
    const int64_t few = std::max<int64_t>(16 / G, 1), others = std::max<int64_t>(total - seqlen, 0);
    if (packed && B > 1 && few * G <= kSplitCols && others <= (B - 1) * few && B * few * Hq < (1 << 24)) r.most = (int)few;
    // The tile kernel.  Splits: as many as fill the workgroup slots (two per compute unit, one at
    // head dim 256) once, at most 16 and of four tiles at least.
    r.row_split = cols <= kTileCols / 2 && d <= 128 ? 2 : 1;
    const int64_t tile_cols = kTileCols / r.row_split, tiles = (cols + tile_cols - 1) / tile_cols;
    // column tiles of packed tokens: at most one that is not full in each sequence
    const int64_t part = r.most ? std::min(B, 1 + others / (few + 1)) : B;
    const int64_t all = std::max<int64_t>(std::min(B * tiles, total * G / tile_cols + part), 1);
    r.tile_cols = (int)tiles, r.items = all;
    const int64_t blocks = Hkv * all, slots = (int64_t)ncu * (d > 128 ? 1 : 2);
    const int64_t longest = (capacity + 4 * tile_rows(d) - 1) / (4 * tile_rows(d));
    const int64_t n = std::min<int64_t>({(slots + blocks / 2) / blocks, 16, longest});
    r.splits = (int)std::max<int64_t>(n, 1);
    if (!r.most) return r;
    cols = few * G;
  }
  const int waves = paged_waves(d, fp8);
  r.nc = cols <= 16 || d > 128 ? 1 : 2;   // (head dim 256: two tiles would not fit the registers)
  r.col_tiles = (int)((cols + 16 * r.nc - 1) / (16 * r.nc));
  r.cols = (int)cols;
  // One workgroup per sequence and KV head, and no second kernel, where that is one round of
  // short ones (1000 rows: 12.9 us, in runs 13.5; 512 workgroups of up to 1500 rows: 41 us, in
  // runs 36).
  // (Of one token: results that are not finite under a mask are the second kernel's.)
  r.direct = !r.most && capacity <= kDirectRows && !packed && seqlen == 1 && B * Hkv * r.col_tiles <= ncu;
  // KV heads of a workgroup, by the rows that its run has at most (measured on 32/8 heads of 128,
  // 8 bits, with 1 / 2 / 4 heads): 4096 x 4 rows 18.7 / 18.5 / 19.8 us, 16 x 8000 43.2 / 41.3 /
  // 42.6, 64 x 2500 54.5 / 45.5 / 46.6, 32 x 32768 206 / 186 / 178.
  r.wave_heads = 1;
  const int64_t run_rows = B * capacity * Hkv / ncu;
  if (!r.direct && Hkv % 2 == 0 && run_rows >= 2 * 1280) r.wave_heads = Hkv % 4 == 0 && run_rows >= 4 * 2048 ? 4 : 2;
  r.unit_rows = 32 * waves / r.wave_heads;   // a step of each wave
  // one run per compute unit (two: decode of 32 x 32768 rows 178 -> 190 us)
  const int64_t most = B * ((capacity + r.unit_rows - 1) / r.unit_rows + 1);
  const int64_t parts = std::min<int64_t>(ncu / (Hkv / r.wave_heads * r.col_tiles), most);
  r.parts = (int)(r.direct ? B : std::max<int64_t>(parts, 1));
  return r;
}

template <class T, bool FP8, int D>
static hipError_t launch_attn_t(PagedAttnParams p, hipStream_t st) {
  if (p.splits) {
    const dim3 tiles((unsigned)(p.tile_blocks + (p.splits > 1 ? 0 : p.rest_blocks)));
    if (D > 128 || p.row_split == 1) hipLaunchKernelGGL((paged_tile_kernel<T, FP8, D, 1>), tiles, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_tile_kernel<T, FP8, (D > 128 ? 128 : D), 2>), tiles, dim3(256), 0, st, p);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && p.splits > 1) {
      const int64_t threads = (int64_t)p.c.total * p.c.Hq * (D / 4);
      hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, p);
      e = hipGetLastError();
    }
    if (e != hipSuccess || !p.c.most) return e;
    p.c.n = p.c.most;   // and the sequences of few tokens
  }
  const dim3 grid((unsigned)(p.parts * (p.c.Hkv / p.wave_heads) * p.col_tiles)), block(paged_waves(D, FP8) * 64);
  constexpr int D2 = D > 128 ? 128 : D;   // (two tiles: up to head dim 128)
  const bool one = p.c.n == 1;
  if (D > 128 || p.nc == 1) {
    if (one) hipLaunchKernelGGL((paged_split_kernel<T, FP8, D, 1, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_split_kernel<T, FP8, D, 1, false>), grid, block, 0, st, p);
  } else {
    if (one) hipLaunchKernelGGL((paged_split_kernel<T, FP8, D2, 2, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_split_kernel<T, FP8, D2, 2, false>), grid, block, 0, st, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.direct) return e;
  const int64_t rows = (p.c.most ? (int64_t)p.c.B * p.c.most : p.c.total) * p.c.Hq;
  if (p.parts / p.c.B < 8)   // (pieces of a sequence, about)
    hipLaunchKernelGGL((paged_combine_kernel<T, FP8, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((paged_combine_kernel<T, FP8, D, 4>), dim3((unsigned)rows), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <int D>
static hipError_t launch_attn_d(const PagedAttnParams& p, hipStream_t st) {
  if (p.c.fp8) return p.c.bf16 ? launch_attn_t<bf16_t, true, D>(p, st) : launch_attn_t<half_t, true, D>(p, st);
  return p.c.bf16 ? launch_attn_t<bf16_t, false, D>(p, st) : launch_attn_t<half_t, false, D>(p, st);
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
