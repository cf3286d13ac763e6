// The 8-bit paged key / value cache: its layout, appending to it with the position rotation, and attention over it.
//
// A page holds P tokens (16, 32 or 64) of one sequence. The pool keeps one record of 2 * P * DH + 16 bytes per (page,
// kv head): the e4m3 codes of the keys, those of the values, then the fp32 scales of the two and a mark (1: all values are 0);
// value = code * scale. A page is quantised once, when its last token arrives, from 16-bit values: until then its tokens live in
// the 16-bit tail, a ring of two pages per (sequence, kv head) addressed by the page's parity. So the codes depend on the tokens
// alone, not on how they arrived, and a sequence can be cut back to any length whose last page is still in the ring.
//
// Inside a page (record and tail alike) the elements of each 16-token group stand in the order in which the m16n8k16
// fragments take them, so that a warp reads a fragment with one vector load per lane from consecutive addresses:
//   keys    [h][r][g][t][e]            token = 8 r + g, dim = h * 4E + t * E + e       (E = min(16, DH / 4))
//   values  [c][g][t][m][r][kh][lo]    token = 8 kh + 2 t + lo, dim = (c * M + m) * 16 + 8 r + g    (M = 2, 1 at DH 16)
// with g = lane / 4 and t = lane % 4.
#pragma once
#include <type_traits>
#include <cuda_fp8.h>
#include "common.cuh"
#include "tc.cuh"

namespace ta {

template <int DH>
struct PageShape {
  static constexpr int E = DH >= 64 ? 16 : DH / 4;  // key elements of one token that a lane holds together
  static constexpr int HG = DH / (4 * E);
  static constexpr int M = DH >= 32 ? 2 : 1;        // 16-dim tiles of the values that a lane holds together
  static constexpr int C = DH / (16 * M);
};

// Offset of an element in its 16-token group (DH * 16 elements), i = token of the group.
template <int DH>
__device__ __forceinline__ int key_offset(int i, int d) {
  using S = PageShape<DH>;
  const int h = d / (4 * S::E), t = (d / S::E) % 4, e = d % S::E;
  return (((h * 2 + (i >> 3)) * 8 + (i & 7)) * 4 + t) * S::E + e;
}
template <int DH>
__device__ __forceinline__ int value_offset(int i, int d) {
  using S = PageShape<DH>;
  const int c = d / (16 * S::M), m = (d / 16) % S::M, r = (d >> 3) & 1, g = d & 7;
  const int kh = i >> 3, t = (i >> 1) & 3, lo = i & 1;
  return ((((c * 8 + g) * 4 + t) * S::M + m) * 2 + r) * 4 + kh * 2 + lo;
}

// The cache of one layer, as every kernel here takes it.
struct PagedCache {
  unsigned char* pool;   // (n_pages, Hkv, record)
  void* tail;            // (B, Hkv, 2 parities, 2 key / value, P * DH) 16-bit
  const int32_t* table;  // (B, max_pages) page of each P tokens
  int64_t table_sb;
  int n_pages, max_pages, Hkv, P;
};

// Sequence b's new rows: rows [start[b], start[b + 1]) at positions pos[b] ... . Returns false (after recording the fault)
// when the numbers do not describe rows of this call: nothing of the sequence is then read or written.
struct NewRows {
  int row0, n, pos;
};
__device__ __forceinline__ bool new_rows(const int32_t* start, const int32_t* pos, int b, int n_rows, int max_new,
                                         const PagedCache& c, int kernel, NewRows& out) {
  const int r0 = start[b], r1 = start[b + 1], p = pos[b];
  out.row0 = r0;
  out.n = r1 - r0;
  out.pos = p;
  if (r0 < 0 || r1 < r0 || r1 > n_rows || r1 - r0 > max_new) {
    if (threadIdx.x == 0) record_error(DEV_INDEX_RANGE, kernel, b, r1 - r0);
    return false;
  }
  if (p < 0 || (int64_t)p + (r1 - r0) > (int64_t)c.max_pages * c.P + (c.P - 1)) {
    if (threadIdx.x == 0) record_error(DEV_POS_RANGE, kernel, b, p);
    return false;
  }
  return true;
}

// What attention reads in place of a page outside the pool: codes 0 and a key scale of NaN, for the rows that see it. A record of
// any page size ends where it ends.
struct alignas(16) OutsideRecord {
  float codes[2 * 64 * 128 / 4], scales[4];
};
static __device__ const OutsideRecord g_outside = {{}, {NAN, 1.f, 0.f, 0.f}};
// The record of a page and kv head; one outside the pool is recorded.
__device__ __forceinline__ const unsigned char* record_of(const PagedCache& c, int page, int h, int rec_bytes, int b) {
  const bool outside = (uint32_t)page >= (uint32_t)c.n_pages;
  if (__builtin_expect(outside, 0)) record_error(DEV_INDEX_RANGE, K_PAGED_ATTN, b, page);
  const unsigned char* rec = c.pool + ((int64_t)page * c.Hkv + h) * rec_bytes;
  return outside ? reinterpret_cast<const unsigned char*>(&g_outside + 1) - rec_bytes : rec;
}

template <int BYTES>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
template <int BYTES>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 16)
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (BYTES == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = w[0];
}

// ------------------------------------------------------------------------------------------------ append
//   y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin   (dims i and i + rot / 2; products and sums rounded one by one in fp32)
// rounded once to the 16-bit type: what the tail holds and what a full page is quantised from.
//   scale = top / 448, code = e4m3(x * (448 / top)), top = the largest magnitude of the page's P x DH values.
// A page whose top is below 2^-100 has codes 0 and scale 1; one that holds an infinity or NaN has codes 0 and scale NaN, so
// that it reads back as NaN.
constexpr int APPEND_THREADS = 128;
constexpr float ZERO_MARK = 1.f;  // beside a record's scales: its values are all 0

struct AppendParams {
  PagedCache c;
  const void *k, *v, *q;
  int64_t k_sr, k_sh, v_sr, v_sh, q_sr, q_sh;
  void* q_out;  // (rows, Hq, DH) contiguous, or null
  const int32_t *start, *pos;
  const float *cosv, *sinv;  // (n_pos, rot / 2)
  int n_pos, rot;
  int n_rows, max_new, Hq;
  int page_ctas;  // CTAs of a sequence that take keys and values; the others rotate queries
};

// Largest magnitude as the bit pattern of the 16-bit type (ordered like the values, infinities and NaN on top).
template <typename T>
__device__ __forceinline__ float bits_value(uint32_t b);
template <>
__device__ __forceinline__ float bits_value<__nv_bfloat16>(uint32_t b) { return __uint_as_float(b << 16); }
template <>
__device__ __forceinline__ float bits_value<__half>(uint32_t b) {
  return __half2float(__ushort_as_half((unsigned short)b));
}

__device__ __forceinline__ uint16_t fp8x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight elements of one row rotated against the eight half_rot further on.
template <typename T>
__device__ __forceinline__ void rotate8(uint4& a, uint4& b, const float* cosv, const float* sinv) {
  float x[8], y[8], c[8], s[8];
  load_vec_f32<T>(reinterpret_cast<const T*>(&a), x);
  load_vec_f32<T>(reinterpret_cast<const T*>(&b), y);
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    ldg_vec_f32<float>(cosv + i, c + i);
    ldg_vec_f32<float>(sinv + i, s + i);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
    y[i] = __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(x[i], s[i]));
    x[i] = u;
  }
  store_vec_from_f32<T>(reinterpret_cast<T*>(&a), x);
  store_vec_from_f32<T>(reinterpret_cast<T*>(&b), y);
}

// 64 positions (64 / P pages) of one (sequence, kv head) per CTA, and CTAs for the rotation of the queries. The rows come
// in 16-byte pieces, eight elements and their partners to a thread; they meet in shared memory, a warp finds the largest
// magnitudes of its 16 tokens, and the codes leave in 16-byte pieces of the page's order. HBM-bound for prompts (4 x 8192
// tokens, 12 heads of 64: 41 us, 6.1 TB/s), launch-bound for single tokens.
constexpr int APPEND_SPAN = 64;

template <typename T, int DH>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(AppendParams p) {
  using S = PageShape<DH>;
  constexpr int PITCH = DH + 8;  // shared rows: a fragment's 8 tokens fall on distinct banks
  extern __shared__ __align__(16) unsigned char append_smem[];
  __shared__ uint32_t tops[2][APPEND_SPAN / 16];
  const int b = blockIdx.y, tid = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  NewRows nr;
  if (!new_rows(p.start, p.pos, b, p.n_rows, p.max_new, p.c, K_PAGED_APPEND, nr) || nr.n == 0) return;
  const int half_rot = p.rot / 2;
  if (p.rot && nr.pos + nr.n > p.n_pos) {
    if (tid == 0) record_error(DEV_POS_RANGE, K_PAGED_APPEND, b, nr.pos + nr.n);
    return;
  }
  const bool vec = half_rot % 8 == 0;  // pairs by eight
  if ((int)blockIdx.x >= p.page_ctas) {
    // ---- queries
    const int cta = blockIdx.x - p.page_ctas, n_cta = gridDim.x - p.page_ctas;
    const T* q = reinterpret_cast<const T*>(p.q);
    T* o = reinterpret_cast<T*>(p.q_out);
    const int pairs = vec ? half_rot / 8 : half_rot;           // pieces (or single elements) with a partner
    const int per = pairs + (vec ? (DH - p.rot) / 8 : DH - p.rot);  // of a row and head
    const int total = nr.n * p.Hq * per;
    for (int id = cta * APPEND_THREADS + tid; id < total; id += n_cta * APPEND_THREADS) {
      const int i = id % per, rh = id / per, h = rh % p.Hq, r = rh / p.Hq;
      const T* src = q + (int64_t)(nr.row0 + r) * p.q_sr + (int64_t)h * p.q_sh;
      T* dst = o + ((int64_t)(nr.row0 + r) * p.Hq + h) * DH;
      const int64_t at = (int64_t)(nr.pos + r) * half_rot;
      if (vec) {
        const int d = i < pairs ? i * 8 : p.rot + (i - pairs) * 8;
        uint4 x = __ldg(reinterpret_cast<const uint4*>(src + d));
        if (i < pairs) {
          uint4 y = __ldg(reinterpret_cast<const uint4*>(src + d + half_rot));
          rotate8<T>(x, y, p.cosv + at + d, p.sinv + at + d);
          *reinterpret_cast<uint4*>(dst + d + half_rot) = y;
        }
        *reinterpret_cast<uint4*>(dst + d) = x;
      } else if (i < pairs) {
        const float c = p.cosv[at + i], s = p.sinv[at + i], x1 = to_f32(src[i]), x2 = to_f32(src[i + half_rot]);
        dst[i] = from_f32<T>(__fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s)));
        dst[i + half_rot] = from_f32<T>(__fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s)));
      } else {
        dst[p.rot + i - pairs] = src[p.rot + i - pairs];
      }
    }
    return;
  }
  // ---- keys and values
  const int P = p.c.P, lp = 31 - __clz(P), h = blockIdx.x % p.c.Hkv;
  const int end = nr.pos + nr.n;
  const int base = (nr.pos / APPEND_SPAN + (int)blockIdx.x / p.c.Hkv) * APPEND_SPAN;  // position of shared row 0
  if (base >= end) return;
  const int f = nr.pos >> lp, last = (end - 1) >> lp;  // first and last page with new tokens
  const int j0 = base >> lp;                           // first page of this CTA
  const int full_end = min(end >> lp << lp, base + APPEND_SPAN) - base;  // rows below this are of full pages
  const int i0 = max(nr.pos - base, 0), i1 = min(end - base, APPEND_SPAN);  // rows with new tokens
  // The last two pages stay in 16 bits. Where the first page has earlier tokens in the tail and the last page is the second
  // after it or later, one of the two may share its slots: then the CTA that reads those tokens writes both, after that.
  const bool old = (nr.pos & (P - 1)) != 0, reader = f >= j0 && f < j0 + (APPEND_SPAN >> lp);
  const int keep = max((last - 1) * P - base, i0);  // rows from here on go to the tail
  const bool keeps = keep < i1 && (!old || reader || last < f + 2);
  T* sk = reinterpret_cast<T*>(append_smem);
  T* sv = sk + APPEND_SPAN * PITCH;
  T* tail = reinterpret_cast<T*>(p.c.tail) + ((int64_t)b * p.c.Hkv + h) * 4 * ((int64_t)P * DH);
  auto tail_k = [&](int page) { return tail + (page & 1) * 2 * ((int64_t)P * DH); };
  const T* kr = reinterpret_cast<const T*>(p.k) + (int64_t)h * p.k_sh;
  const T* vr = reinterpret_cast<const T*>(p.v) + (int64_t)h * p.v_sh;
  constexpr int VPR = DH / 8;
  // rows [r0, r1) of the span at position `from` into shared memory, keys rotated
  auto load_rows = [&](int from, int r0, int r1) {
    const int64_t row = (int64_t)nr.row0 + from - nr.pos;
    if (!half_rot) {
#pragma unroll 4
      for (int id = tid; id < (r1 - r0) * VPR; id += APPEND_THREADS) {
        const int i = r0 + id / VPR, d = id % VPR * 8;
        *reinterpret_cast<uint4*>(sk + i * PITCH + d) = __ldg(reinterpret_cast<const uint4*>(kr + (row + i) * p.k_sr + d));
        *reinterpret_cast<uint4*>(sv + i * PITCH + d) = __ldg(reinterpret_cast<const uint4*>(vr + (row + i) * p.v_sr + d));
      }
      return;
    }
    if (vec) {
      const int pairs = half_rot / 8, per = VPR - pairs;
#pragma unroll 4
      for (int id = tid; id < (r1 - r0) * per; id += APPEND_THREADS) {
        const int i = r0 + id / per, c = id % per;
        const int d = c < pairs ? c * 8 : p.rot + (c - pairs) * 8;
        const T* src = kr + (row + i) * p.k_sr;
        uint4 x = __ldg(reinterpret_cast<const uint4*>(src + d));
        if (c < pairs) {
          uint4 y = __ldg(reinterpret_cast<const uint4*>(src + d + half_rot));
          const int64_t at = (int64_t)(from + i) * half_rot + d;
          rotate8<T>(x, y, p.cosv + at, p.sinv + at);
          *reinterpret_cast<uint4*>(sk + i * PITCH + d + half_rot) = y;
        }
        *reinterpret_cast<uint4*>(sk + i * PITCH + d) = x;
      }
    } else {
      for (int id = tid; id < (r1 - r0) * (DH - half_rot); id += APPEND_THREADS) {
        const int i = r0 + id / (DH - half_rot), d = id % (DH - half_rot);
        const T* src = kr + (row + i) * p.k_sr;
        if (d < half_rot) {
          const int64_t at = (int64_t)(from + i) * half_rot + d;
          const float c = p.cosv[at], s = p.sinv[at], x1 = to_f32(src[d]), x2 = to_f32(src[d + half_rot]);
          sk[i * PITCH + d] = from_f32<T>(__fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s)));
          sk[i * PITCH + d + half_rot] = from_f32<T>(__fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s)));
        } else {
          sk[i * PITCH + d + half_rot] = src[d + half_rot];
        }
      }
    }
#pragma unroll 4
    for (int id = tid; id < (r1 - r0) * VPR; id += APPEND_THREADS) {
      const int i = r0 + id / VPR, d = id % VPR * 8;
      *reinterpret_cast<uint4*>(sv + i * PITCH + d) = __ldg(reinterpret_cast<const uint4*>(vr + (row + i) * p.v_sr + d));
    }
  };
  // ... and from there into the tail
  auto keep_rows = [&](int from, int r0, int r1) {
    for (int id = tid; id < (r1 - r0) * DH; id += APPEND_THREADS) {
      const int r = r0 + id / DH, d = id % DH, i = (from + r) & (P - 1);
      T* ok = tail_k((from + r) >> lp) + (i >> 4) * 16 * DH;
      ok[key_offset<DH>(i & 15, d)] = sk[r * PITCH + d];
      ok[(int64_t)P * DH + value_offset<DH>(i & 15, d)] = sv[r * PITCH + d];
    }
  };
  if (full_end > i0 || keeps) load_rows(base, i0, i1);
  if (reader && old && ((f + 1) << lp) <= end) {  // the first page's earlier tokens
    const T* ok = tail_k(f);
    const int r0 = (f << lp) - base;
    for (int id = tid; id < (nr.pos & (P - 1)) * DH; id += APPEND_THREADS) {
      const int i = id / DH, d = id % DH;
      sk[(r0 + i) * PITCH + d] = ok[(i >> 4) * 16 * DH + key_offset<DH>(i & 15, d)];
      sv[(r0 + i) * PITCH + d] = ok[(int64_t)P * DH + (i >> 4) * 16 * DH + value_offset<DH>(i & 15, d)];
    }
  }
  __syncthreads();
  if (keeps) keep_rows(base, keep, i1);
  // ---- full pages: rows [g0 * 16, full_end), whole groups of 16 tokens
  const int g0 = max((f << lp) - base, 0) >> 4, g1 = full_end >> 4;
  if (g1 <= g0) return;
  {
    const int warp = tid >> 5, lane = tid & 31;
    if (warp >= g0 && warp < g1) {
      uint32_t mk = 0, mv = 0;
      for (int id = lane; id < 16 * VPR; id += 32) {
        const int at = (warp * 16 + id / VPR) * PITCH + (id % VPR) * 8;
        const uint4 a = *reinterpret_cast<const uint4*>(sk + at), w = *reinterpret_cast<const uint4*>(sv + at);
        const uint32_t ka[4] = {a.x, a.y, a.z, a.w}, va[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          mk = max(mk, max(ka[x] & 0x7fffu, (ka[x] >> 16) & 0x7fffu));
          mv = max(mv, max(va[x] & 0x7fffu, (va[x] >> 16) & 0x7fffu));
        }
      }
      mk = __reduce_max_sync(0xffffffffu, mk);
      mv = __reduce_max_sync(0xffffffffu, mv);
      if (lane == 0) {
        tops[0][warp] = mk;
        tops[1][warp] = mv;
      }
    }
  }
  __syncthreads();
  const int gpp = P >> 4;  // groups of a page
#pragma unroll 1
  for (int pg = g0; pg < g1; pg += gpp) {
    const int j = (base >> lp) + (pg >> (lp - 4));
    const int phys = p.c.table[b * p.c.table_sb + j];
    if (phys < 0 || phys >= p.c.n_pages) {
      if (tid == 0) record_error(DEV_INDEX_RANGE, K_PAGED_APPEND, b, phys);
      continue;
    }
    float mul[2], scale[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t bits = 0;
      for (int g = 0; g < gpp; ++g) bits = max(bits, tops[x][pg + g]);
      const float top = bits_value<T>(bits);
      const bool odd = !(top <= 3.402823466e38f), tiny = top < 7.888609052e-31f;  // 2^-100
      mul[x] = odd || tiny ? 0.f : __fdiv_rn(448.f, top);
      scale[x] = odd ? __int_as_float(0x7fc00000) : (tiny ? 1.f : __fdiv_rn(top, 448.f));
    }
    unsigned char* rec = p.c.pool + ((int64_t)phys * p.c.Hkv + h) * (2 * P * DH + 16);
    if (tid == 0)  // (codes are 0 below 2^-100 alone: the marked pages have scale 1)
      *reinterpret_cast<float4*>(rec + 2 * P * DH) =
          make_float4(scale[0], scale[1], mul[1] == 0.f && scale[1] == 1.f ? ZERO_MARK : 0.f, 0.f);
    // a page with a non-finite element has codes 0 (0 * NaN would not be)
    const bool zk = mul[0] == 0.f, zv = mul[1] == 0.f;
    for (int id = tid; id < P * DH / S::E; id += APPEND_THREADS) {
      // keys: E consecutive dims of one token
      const int t = id % 4, g = id / 4 % 8, r = id / 32 % 2, hg = id / 64 % S::HG, grp = id / (64 * S::HG);
      const T* a = sk + ((pg + grp) * 16 + r * 8 + g) * PITCH + (hg * 4 + t) * S::E;
      uint32_t w[S::E / 4];
#pragma unroll
      for (int e = 0; e < S::E / 4; ++e) {
        uint32_t two[2];
        load_words<8>(a + e * 4, two);
        w[e] = zk ? 0u
                  : fp8x2(bits_value<T>(two[0] & 0xffffu) * mul[0], bits_value<T>(two[0] >> 16) * mul[0]) |
                        ((uint32_t)fp8x2(bits_value<T>(two[1] & 0xffffu) * mul[0], bits_value<T>(two[1] >> 16) * mul[0]) << 16);
      }
      store_words<S::E>(rec + (int64_t)id * S::E, w);
    }
    for (int id = tid; id < P * DH / (8 * S::M); id += APPEND_THREADS) {
      // values: 2 M dims (8 apart) of 4 tokens
      const int t = id % 4, g = id / 4 % 8, c = id / 32 % S::C, grp = id / (32 * S::C);
      const T* a = sv + ((pg + grp) * 16 + 2 * t) * PITCH + c * S::M * 16 + g;
      uint32_t w[2 * S::M];
#pragma unroll
      for (int x = 0; x < 2 * S::M; ++x) {
        const T* v0 = a + x * 8;
        w[x] = zv ? 0u
                  : fp8x2(to_f32(v0[0]) * mul[1], to_f32(v0[PITCH]) * mul[1]) |
                        ((uint32_t)fp8x2(to_f32(v0[8 * PITCH]) * mul[1], to_f32(v0[9 * PITCH]) * mul[1]) << 16);
      }
      store_words<8 * S::M>(rec + P * DH + (int64_t)id * 8 * S::M, w);
    }
  }
  if (reader && old && last >= f + 2) {
    // later pages of other CTAs into the tail (the earlier tokens have been read); the first page is full then, so that no
    // thread has left above
    const int from = max((last - 1) << lp, base + APPEND_SPAN);
    for (int span = from / APPEND_SPAN * APPEND_SPAN; span < end; span += APPEND_SPAN) {
      const int r0 = max(from - span, 0), r1 = min(end - span, APPEND_SPAN);
      __syncthreads();
      load_rows(span, r0, r1);
      __syncthreads();
      keep_rows(span, r0, r1);
    }
  }
}

// ------------------------------------------------------------------------------------------------ attention
// out[r] = sum_t softmax_t(scale q_r . K_t) V_t over the positions t <= pos + i of query i (and t > pos + i - window).
// Rows of a (sequence, kv head): query i, head gq of the group -> row i * group + gq. A warp takes 8 NT rows as the N side of
// mma.m16n8k16 and the keys (S^T = K Q^T) or the head dims (O^T = V^T P^T) as the M side, so that one key or value fragment
// serves every row and a lone row costs one n-tile.
//  * codes go to f16 exactly; q is scaled by a power of two per row (undone in the score's factor; see finish) so that bf16
//    rows fit f16 as well; the products are exact and the sums fp32.
//  * the value scale joins the weight: w_t = exp2(s_t + log2 vs - ref), with the running reference taken over s + log2 vs, so
//    that every w stays in f16's range (at most 2^12); the denominator adds w / vs in fp32. w is rounded to f16 (2^-11
//    relative, 2^-25 of 1 below 2^-14) for the product, the denominator takes it unrounded.
//  * the open page is read in 16 bits from the tail, in the same element order, with the 16-bit type's own mma.
constexpr float ATTN_SHIFT = 12.f;

struct AttnParams {
  PagedCache c;
  const void* q;
  int64_t q_sr, q_sh;
  const int32_t *start, *pos;
  int B, n_rows, max_new, Hq;
  float scale;
  int window;  // 0 = the whole prefix
  void* out;
  int64_t o_sr, o_sh;
  float* lse;  // (rows, Hq) or null
  int probe;   // PROBE: the warp (split form) or CTA (tile form) whose first wait runs out
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    mma_f16(d, a, b0, b1);
  else
    mma_bf16(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// four e4m3 codes -> two f16x2
__device__ __forceinline__ void codes_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {  // results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// A page whose values are all 0 (or below 2^-100) stores scale 1, whatever the pages beside it hold. Taken as it stands it would
// lift the reference 2^20 and more above pages of small values, whose weights then fall among f16's subnormals (values of
// 1e-6 behind such a page: 7 % off). Its codes are 0, so any scale will do: 2^-64 lets its tokens weigh what their scores say
// while those of values between 2^-75 and 2^49 keep their bits. (The open page needs none: it is the last that a running
// softmax takes, and what came before it is in fp32 by then.) sc: the record's two scales and its mark.
__device__ __forceinline__ void value_factors(const float4& sc, float& lv, float& iv) {
  const float vs = sc.z == ZERO_MARK ? 5.421010862427522e-20f : sc.y;
  lv = log2_fast(vs);
  iv = rcp_fast(vs);
}
// The rows of one tile: query fragments and what the masks and scores need, per lane for its two columns of each n-tile.
template <typename T, int DH, int NT>
struct RowTile {
  using S = PageShape<DH>;
  uint32_t qf[DH / 16][NT][2];  // f16, scaled per row
  float cs[NT][2];              // score factor of the row, positive: |scale| * log2(e) / (its power of two)
  int qpos[NT][2];              // position of the row's query; -1: no such row

  // The rows' elements as stored, in fragment order: fetched early, turned into fragments by finish.
  struct Raw {
    uint32_t w[NT][DH / 8];
  };

  // row0: first row of the tile; R rows in all (n queries x group heads)
  static __device__ __forceinline__ void fetch(const AttnParams& p, int q_row0, int h, int group, int row0, int R, Raw& raw) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int rr = row0 + nt * 8 + g;
      const bool live = rr < R;
      const T* src = reinterpret_cast<const T*>(p.q);
      if (live) src += (int64_t)(q_row0 + rr / group) * p.q_sr + (int64_t)(h * group + rr % group) * p.q_sh;
#pragma unroll
      for (int hg = 0; hg < S::HG; ++hg)
#pragma unroll
        for (int e = 0; e < S::E; e += 4) {
          uint32_t w[2] = {0u, 0u};
          if (live) load_words<8>(src + hg * 4 * S::E + t * S::E + e, w);
          raw.w[nt][(hg * S::E + e) / 2] = w[0];
          raw.w[nt][(hg * S::E + e) / 2 + 1] = w[1];
        }
    }
  }

  __device__ __forceinline__ void finish(const AttnParams& p, int pos, int group, int row0, int R, const Raw& raw) {
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < DH / 8; ++i)
        top = fmaxf(top, fmaxf(fabsf(bits_value<T>(raw.w[nt][i] & 0xffffu)), fabsf(bits_value<T>(raw.w[nt][i] >> 16))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^ex * top in [2^7, 2^8): exact down to 2^-21 of the row's largest element, and within 2^-32 of it below (fp32 sums lose
      // 2^-24). Not higher: bf16 keys of the open page come as they are, and 2^15 times those of 2^110 left fp32's range.
      const int ex = min(7 + 127 - (int)(__float_as_uint(top) >> 23), 120);
      // the sign of the scale joins the row; at scale 0 the row is 0
      const float up = p.scale == 0.f ? 0.f : copysignf(__int_as_float((ex + 127) << 23), p.scale);
#pragma unroll
      for (int i = 0; i < DH / 8; ++i)
        qf[i / 2][nt][i & 1] =
            pack2<__half>(bits_value<T>(raw.w[nt][i] & 0xffffu) * up, bits_value<T>(raw.w[nt][i] >> 16) * up);
      const float f = p.scale == 0.f ? 1.f : fabsf(p.scale) * 1.4426950408889634f * __int_as_float((127 - ex) << 23);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cs[nt][i] = __shfl_sync(0xffffffffu, f, (2 * t + i) * 4);
        const int col = row0 + nt * 8 + 2 * t + i;
        qpos[nt][i] = col < R ? pos + col / group : -1;
      }
    }
  }
};

// Running softmax of a warp: reference (log2 units, uniform over the 8 lanes of a column), denominator (each lane its
// own tokens' part), numerator O^T.
template <int DH, int NT>
struct SoftState {
  float m[NT][2], l[NT][2], o[DH / 16][NT][4];
  __device__ __forceinline__ void clear(float sum = 0.f) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = sum;
#pragma unroll
      for (int x = 0; x < DH / 16; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[x][nt][i] = 0.f;
    }
  }
};

// Scores -> weights for TG 16-token groups, in place: s holds the raw sums. ks / lv / iv: per group the key scale, log2 of the
// value scale and its inverse. tok0: position of the first token; tokens from `limit` on are not the unit's. The factors
// are positive, so that the maximum is taken over the raw sums.
template <typename T, int DH, int NT, int TG>
__device__ __forceinline__ void soft_step(const RowTile<T, DH, NT>& rt, SoftState<DH, NT>& st, float (&s)[TG][NT][4],
                                          const float (&ks)[TG], const float (&lv)[TG], const float (&iv)[TG], int tok0,
                                          int limit, int window, bool mask) {
  const int g = (threadIdx.x & 31) >> 2;
  uint32_t gone[NT];  // masked elements, bit x * 4 + i
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) gone[nt] = 0u;
  if (mask) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int last = min(rt.qpos[nt][i], limit - 1), first = window > 0 ? rt.qpos[nt][i] - window + 1 : 0;
#pragma unroll
        for (int x = 0; x < TG; ++x)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int tok = tok0 + x * 16 + r * 8 + g;
            if (tok > last || tok < first) {
              s[x][nt][r * 2 + i] = -INFINITY;
              gone[nt] |= 1u << (x * 4 + r * 2 + i);
            }
          }
      }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int x = 0; x < TG; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        top[i] = fmaxf(top[i], fmaf(fmaxf(s[x][nt][i], s[x][nt][i + 2]), ks[x] * rt.cs[nt][i], lv[x]));
    float ref[2], fac[2];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 4));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 8));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
      const float mn = fmaxf(st.m[nt][i], top[i]);
      fac[i] = mn == st.m[nt][i] ? 1.f : exp2_fast(st.m[nt][i] - mn);
      moved |= mn != st.m[nt][i];
      st.m[nt][i] = mn;
      ref[i] = mn == -INFINITY ? 0.f : mn - ATTN_SHIFT;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) st.l[nt][i] *= fac[i];
#pragma unroll
      for (int x = 0; x < DH / 16; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[x][nt][i] *= fac[i & 1];
    }
#pragma unroll
    for (int x = 0; x < TG; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[x][nt][i] = exp2_fast(fmaf(s[x][nt][i], ks[x] * rt.cs[nt][i & 1], lv[x] - ref[i & 1]));
    if (mask) {  // a masked token weighs 0 whatever its page's scales are
#pragma unroll
      for (int x = 0; x < TG; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (gone[nt] >> (x * 4 + i) & 1u) s[x][nt][i] = 0.f;
    }
#pragma unroll
    for (int x = 0; x < TG; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float sum = s[x][nt][i] + s[x][nt][i + 2];
        st.l[nt][i] += sum == 0.f ? 0.f : sum * iv[x];
      }
  }
}

// One unit of TG 16-token groups of 8-bit pages: kp / vp per group its key and value codes.
template <typename T, int DH, int NT, int TG>
__device__ __forceinline__ void attend_codes(const RowTile<T, DH, NT>& rt, SoftState<DH, NT>& st,
                                             const unsigned char* const (&kp)[TG], const unsigned char* const (&vp)[TG],
                                             const float (&ks)[TG], const float (&lv)[TG], const float (&iv)[TG],
                                             int tok0, int limit, int window, bool mask) {
  using S = PageShape<DH>;
  const int lane = threadIdx.x & 31;
  float s[TG][NT][4];
#pragma unroll
  for (int x = 0; x < TG; ++x)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][nt][i] = 0.f;
#pragma unroll
  for (int hg = 0; hg < S::HG; ++hg)
#pragma unroll
    for (int x = 0; x < TG; ++x) {
      uint32_t w0[S::E / 4], w1[S::E / 4];
      load_words<S::E>(kp[x] + (hg * 2 * 32 + lane) * S::E, w0);
      load_words<S::E>(kp[x] + ((hg * 2 + 1) * 32 + lane) * S::E, w1);
#pragma unroll
      for (int e = 0; e < S::E / 4; ++e) {
        uint32_t a[4];
        codes_f16x4(w0[e], a[0], a[2]);
        codes_f16x4(w1[e], a[1], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(s[x][nt], a, rt.qf[hg * (S::E / 4) + e][nt][0], rt.qf[hg * (S::E / 4) + e][nt][1]);
      }
    }
  soft_step<T, DH, NT, TG>(rt, st, s, ks, lv, iv, tok0, limit, window, mask);
  uint32_t pf[TG][NT][2];
#pragma unroll
  for (int x = 0; x < TG; ++x)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      pf[x][nt][0] = transpose8x8(pack2<__half>(s[x][nt][0], s[x][nt][1]));
      pf[x][nt][1] = transpose8x8(pack2<__half>(s[x][nt][2], s[x][nt][3]));
    }
#pragma unroll
  for (int x = 0; x < TG; ++x)
#pragma unroll
    for (int c = 0; c < S::C; ++c) {
      uint32_t w[2 * S::M];
      load_words<8 * S::M>(vp[x] + (c * 32 + lane) * 8 * S::M, w);
#pragma unroll
      for (int m = 0; m < S::M; ++m) {
        uint32_t a[4];
        codes_f16x4(w[2 * m], a[0], a[2]);
        codes_f16x4(w[2 * m + 1], a[1], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(st.o[c * S::M + m][nt], a, pf[x][nt][0], pf[x][nt][1]);
      }
    }
}

// A query fragment in the tail's type: the power of two keeps bf16 rows exact as well.
template <typename T>
__device__ __forceinline__ uint32_t as_type(uint32_t f16x2) {
  if constexpr (std::is_same<T, __half>::value) return f16x2;
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&f16x2));
  return pack2<T>(f.x, f.y);
}

// Infinities and NaN among the open page's values. In the product a masked token's weight of 0 would make them NaN for every row
// of the tile, so they stay out of it, and the rows that see their tokens get them at the end, when the output is written.
// odd2: bit 15 (31) of two elements that are one: above the largest finite magnitude, one step of the exponent's last place
// carries into it. finite2: the elements with those taken out (0).
template <typename T>
__device__ __forceinline__ uint32_t odd2(uint32_t w) {
  return ((w & 0x7fff7fffu) + (std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  return w & ~((odd2<T>(w) >> 15) * 0xffffu);
}
// Takes them out of n 16-byte pieces in shared memory (the warp's own); whether there were any.
template <typename T>
__device__ __forceinline__ bool clean_values(unsigned char* v, int n) {
  const int lane = threadIdx.x & 31;
  uint32_t odd = 0u;
#pragma unroll 4
  for (int i = lane; i < n; i += 32) {
    const uint4 w = reinterpret_cast<const uint4*>(v)[i];
    odd |= odd2<T>(w.x) | odd2<T>(w.y) | odd2<T>(w.z) | odd2<T>(w.w);
  }
  if (__builtin_expect(!__any_sync(0xffffffffu, odd != 0u), 1)) return false;
#pragma unroll 1
  for (int i = lane; i < n; i += 32) {
    uint4 w = reinterpret_cast<uint4*>(v)[i];
    w.x = finite2<T>(w.x); w.y = finite2<T>(w.y); w.z = finite2<T>(w.z); w.w = finite2<T>(w.w);
    reinterpret_cast<uint4*>(v)[i] = w;
  }
  fence_proxy_async_smem();  // the place is filled by a bulk copy next
  __syncwarp();
  return true;
}
// Adds those of the open page (values tv; positions from `first` on) to a row that sees the positions [from, to), dims d0,
// d0 + step, ... below d1.
template <typename T, int DH>
__device__ __noinline__ void add_odd(const T* tv, int first, int from, int to, int d0, int d1, int step, T* out) {
  for (int at = max(from, first); at < to; ++at) {
    const int i = at - first;
    for (int d = d0; d < d1; d += step) {
      const float v = to_f32(tv[(i >> 4) * 16 * DH + value_offset<DH>(i & 15, d)]);
      if (!(fabsf(v) <= 3.402823466e38f)) out[d] = from_f32<T>(to_f32(out[d]) + v);
    }
  }
}
// The values of the open page of sequence b and kv head h: page n_full.
template <typename T, int DH>
__device__ __forceinline__ const T* open_values(const PagedCache& c, int b, int h, int n_full) {
  return reinterpret_cast<const T*>(c.tail) + ((((int64_t)b * c.Hkv + h) * 2 + (n_full & 1)) * 2 + 1) * ((int64_t)c.P * DH);
}

// TG 16-token groups of the open page, 16-bit elements in the same order. len: tokens the sequence holds; later slots of
// the page hold anything and are masked in the scores and zeroed in the values. CLEAN: the values hold no infinity or NaN;
// otherwise those are left out here, and odd is set.
template <typename T, int DH, int NT, int TG, bool CLEAN>
__device__ __forceinline__ void attend_tail(const RowTile<T, DH, NT>& rt, SoftState<DH, NT>& st, const T* kp, const T* vp,
                                            int tok0, int len, int window, uint32_t& odd) {
  using S = PageShape<DH>;
  const int lane = threadIdx.x & 31, t = lane & 3;
  float s[TG][NT][4];
#pragma unroll
  for (int x = 0; x < TG; ++x)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][nt][i] = 0.f;
#pragma unroll
  for (int hg = 0; hg < S::HG; ++hg)
#pragma unroll
    for (int e = 0; e < S::E / 4; ++e) {
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        b0[nt] = as_type<T>(rt.qf[hg * (S::E / 4) + e][nt][0]);
        b1[nt] = as_type<T>(rt.qf[hg * (S::E / 4) + e][nt][1]);
      }
#pragma unroll
      for (int x = 0; x < TG; ++x) {
        uint32_t w0[2], w1[2];
        load_words<8>(kp + x * 16 * DH + (hg * 2 * 32 + lane) * S::E + e * 4, w0);
        load_words<8>(kp + x * 16 * DH + ((hg * 2 + 1) * 32 + lane) * S::E + e * 4, w1);
        const uint32_t a[4] = {w0[0], w1[0], w0[1], w1[1]};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16<T>(s[x][nt], a, b0[nt], b1[nt]);
      }
    }
  float one[TG], zero[TG];
#pragma unroll
  for (int x = 0; x < TG; ++x) {
    one[x] = 1.f;
    zero[x] = 0.f;
  }
  soft_step<T, DH, NT, TG>(rt, st, s, one, zero, one, tok0, len, window, true);
#pragma unroll
  for (int x = 0; x < TG; ++x) {
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      pf[nt][0] = transpose8x8(pack2<T>(s[x][nt][0], s[x][nt][1]));
      pf[nt][1] = transpose8x8(pack2<T>(s[x][nt][2], s[x][nt][3]));
    }
    const int k0 = tok0 + x * 16 + 2 * t;
    const uint32_t keep0 = (k0 < len ? 0xffffu : 0u) | (k0 + 1 < len ? 0xffff0000u : 0u);
    const uint32_t keep1 = (k0 + 8 < len ? 0xffffu : 0u) | (k0 + 9 < len ? 0xffff0000u : 0u);
#pragma unroll
    for (int c = 0; c < S::C; ++c) {
      uint32_t w[4 * S::M];
      load_words<16 * S::M>(vp + x * 16 * DH + (c * 32 + lane) * 8 * S::M, w);
      if constexpr (!CLEAN) {
#pragma unroll
        for (int i = 0; i < 4 * S::M; ++i) {
          odd |= odd2<T>(w[i]);
          w[i] = finite2<T>(w[i]);
        }
      }
#pragma unroll
      for (int m = 0; m < S::M; ++m) {
        const uint32_t a[4] = {w[4 * m] & keep0, w[4 * m + 2] & keep0, w[4 * m + 1] & keep1, w[4 * m + 3] & keep1};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16<T>(st.o[c * S::M + m][nt], a, pf[nt][0], pf[nt][1]);
      }
    }
  }
}

// A (row tile, kv head, sequence) per CTA: its 4 warps take the 64-token units in turn, each with its own running softmax,
// and the four states are joined in shared memory.
constexpr int ATTN_WARPS = 4;

template <int DH, int NT>
__host__ __device__ constexpr int attn_smem_bytes() {
  return ATTN_WARPS * 8 * NT * (DH + 4) * 4 + ATTN_WARPS * 8 * NT * 2 * 4;
}

template <typename T, int DH, int NT>
__global__ void __launch_bounds__(ATTN_WARPS * 32) paged_attn_kernel(AttnParams p) {
  constexpr int ROWS = 8 * NT, PITCH = DH + 4;
  extern __shared__ __align__(16) unsigned char attn_smem[];
  float* so = reinterpret_cast<float*>(attn_smem);       // (warp, row, DH)
  float* sm = so + ATTN_WARPS * ROWS * PITCH;            // (warp, row)
  float* sl = sm + ATTN_WARPS * ROWS;
  const int b = blockIdx.z, h = blockIdx.y, row0 = blockIdx.x * ROWS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  NewRows nr;
  if (!new_rows(p.start, p.pos, b, p.n_rows, p.max_new, p.c, K_PAGED_ATTN, nr)) return;
  const int group = p.Hq / p.c.Hkv, R = nr.n * group, P = p.c.P;
  if (row0 >= R) return;
  const int len = nr.pos + nr.n, n_full = len / P;
  const int qlo = nr.pos + row0 / group, qhi = nr.pos + (min(R, row0 + ROWS) - 1) / group;
  const int lo = p.window > 0 ? max(0, qlo - p.window + 1) : 0;
  const int p0 = lo / P, p1 = min(n_full, qhi / P + 1), limit = p1 * P;
  const int per = 64 / P;
  RowTile<T, DH, NT> rt;
  {
    typename RowTile<T, DH, NT>::Raw raw;
    rt.fetch(p, nr.row0, h, group, row0, R, raw);
    rt.finish(p, nr.pos, group, row0, R, raw);
  }
  SoftState<DH, NT> st;
  st.clear();
  const int32_t* tab = p.c.table + b * p.c.table_sb;
  const int rec_bytes = 2 * P * DH + 16;
  uint32_t odd = 0u;
  for (int u = p0 + warp * per; u < p1; u += ATTN_WARPS * per) {
    const unsigned char *kp[4], *vp[4];
    float ks[4], lv[4], iv[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int pg = min(u + x * 16 / P, p1 - 1);
      const unsigned char* rec = record_of(p.c, tab[pg], h, rec_bytes, b);
      kp[x] = rec + (x * 16 % P) * DH;
      vp[x] = kp[x] + P * DH;
      const float4 sc = *reinterpret_cast<const float4*>(rec + 2 * P * DH);
      ks[x] = sc.x;
      value_factors(sc, lv[x], iv[x]);
    }
    const int tok0 = u * P;
    const bool mask = tok0 + 63 > min(qlo, limit - 1) || (p.window > 0 && tok0 <= qhi - p.window);
    attend_codes<T, DH, NT, 4>(rt, st, kp, vp, ks, lv, iv, tok0, limit, p.window, mask);
  }
  if (n_full * P <= qhi) {
    const T* tk = reinterpret_cast<const T*>(p.c.tail) +
                  ((((int64_t)b * p.c.Hkv + h) * 2 + (n_full & 1)) * 2) * ((int64_t)P * DH);
    for (int x = warp; n_full * P + x * 16 <= qhi; x += ATTN_WARPS)
      attend_tail<T, DH, NT, 1, false>(rt, st, tk + x * 16 * DH, tk + (int64_t)P * DH + x * 16 * DH, n_full * P + x * 16, len,
                                       p.window, odd);
  }
  // join the warps
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float l = st.l[nt][i];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int col = nt * 8 + 2 * t + i;
      if (g == 0) {
        sm[warp * ROWS + col] = st.m[nt][i];
        sl[warp * ROWS + col] = l;
      }
#pragma unroll
      for (int x = 0; x < DH / 16; ++x) {
        so[(warp * ROWS + col) * PITCH + x * 16 + g] = st.o[x][nt][i];
        so[(warp * ROWS + col) * PITCH + x * 16 + 8 + g] = st.o[x][nt][i + 2];
      }
    }
  odd = __syncthreads_or(odd != 0u);
  for (int id = tid; id < ROWS * DH; id += ATTN_WARPS * 32) {
    const int col = id / DH, d = id % DH, rr = row0 + col;
    if (rr >= R) break;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < ATTN_WARPS; ++w) m = fmaxf(m, sm[w * ROWS + col]);
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < ATTN_WARPS; ++w) {
      const float f = sm[w * ROWS + col] == -INFINITY ? 0.f : exp2f(sm[w * ROWS + col] - m);
      if (f == 0.f && m != -INFINITY && sl[w * ROWS + col] == 0.f) continue;
      L += sl[w * ROWS + col] * f;
      o += so[(w * ROWS + col) * PITCH + d] * f;
    }
    const int64_t row = nr.row0 + rr / group;
    const int hq = h * group + rr % group;
    T* out = reinterpret_cast<T*>(p.out) + row * p.o_sr + hq * p.o_sh;
    out[d] = from_f32<T>(L == 0.f ? 0.f : o / L);
    if (odd) {
      const int qp = nr.pos + rr / group;
      add_odd<T, DH>(open_values<T, DH>(p.c, b, h, n_full), n_full * P, p.window > 0 ? qp - p.window + 1 : 0, min(len, qp + 1), d,
                     d + 1, 1, out);
    }
    if (p.lse && d == 0)
      p.lse[row * p.Hq + hq] = L == 0.f ? -INFINITY : (m - ATTN_SHIFT + log2f(L)) * 0.69314718055994531f;
  }
}

// ------------------------------------------------------------------------------------------------ attention, few rows
// At most 32 rows per (sequence, kv head): the cache's bytes bound it. An item is a (sequence, kv head); its units are
// runs of 64 tokens of full pages, then of 32 tokens of the open page. The units of all items, in order, are shared out
// evenly over the warps of one resident grid, whatever the lengths are: a warp takes a run of units that may end one item and
// begin another. Each warp keeps its own ring of units in shared memory, filled by bulk copies (a record of a full page is
// one copy, scales included), so the only waits are for its own copies.
// An item that one warp holds whole is written out at once; of the others each warp leaves its state (maximum, sum,
// numerator) in the workspace, and the warp that comes last (a counter per item), or its CTA, joins them in order. The
// counters are left at zero.
template <int DH, int NT>
struct SplitShape {
  // Eight warps' rings, two units ahead of the one at work, fill the shared memory at 8 KB a unit.
  static constexpr int UT = DH == 128 ? 32 : 64;     // tokens of a unit of full pages
  static constexpr int TT = UT / 2;                  // tokens of a unit of the open page (16 bits)
  static constexpr int STAGE = 2 * UT * DH + UT;     // codes, and 16 bytes of scales for up to UT / 16 records
  static constexpr int NS = 3;
  static constexpr int WARPS = 8;
  static constexpr int STATE = 8 * NT * DH + 16 * NT;  // floats: numerator fragments, then (maximum, sum) per row
  static constexpr int BAR_BYTES = WARPS * NS * 8;
  static constexpr int RING = WARPS * NS * STAGE;
};

// Units per warp while warps are plenty: fewer spread more, but have more parts to join (one sequence of 4096, 12 heads:
// 12.3 us with 1, 10.9 with 2, 11.7 with 3).
constexpr int SPLIT_MIN_UNITS = 2;
// An item's own cost, in units (its queries' loads, its output or state): without it a warp whose run is many short sequences
// comes last (64 uneven sequences, one of them a single token: 67 us without it, 64.5 with; windows
// of five rows: 53.8 us with 1, 51.3 with 2 to 4)
constexpr int SPLIT_ITEM_COST = 2;
// Bytes of an item's states up to which the warp that comes last joins them by itself, on the spot, while the others stream;
// the end of a kernel that joins late costs 2 to 7 us at any size. In us, by the last warp / late: 24 parts of 8 rows of head
// dim 64 12.4 / 14.4, 98 parts of one row 18.1 / 17.0, 148 of 8 rows 30.5 / 18.6; of head dim 128, 18 parts 98.8 / 106, 37
// parts 56.5 / 58.6, 46 parts 20.5 / 16.5, 148 parts 57.4 / 28.8; of 32 dims, 148 parts 26.7 / 26.6. States of more than 8
// vectors a lane are always joined late: one warp does not hold two of them.
constexpr int SPLIT_SPOT_BYTES = 176 << 10;
template <int DH, int NT>
constexpr bool split_spot() {
  return DH / 16 * NT <= 8;
}
constexpr int SPLIT_MAX_BATCH = 2048;  // sequences whose geometry is kept in shared memory (12 bytes each)

// The units of one item.
struct Item {
  int pos, n, row0;
  int len, p0, p1;    // tokens held; full pages [p0, p1)
  int nu8, units;     // units of full pages, of all
};
template <int UT>
__device__ __forceinline__ Item item_of(int row0, int n, int pos, int lp, int window) {
  Item it;
  it.row0 = row0;
  it.n = n;
  it.pos = pos;
  it.len = pos + n;
  it.p1 = it.len >> lp;
  it.p0 = window > 0 ? max(0, pos - window + 1) >> lp : 0;
  it.nu8 = (((it.p1 - it.p0) << lp) + UT - 1) / UT;
  it.units = n > 0 ? it.nu8 + (it.len - (it.p1 << lp) + UT / 2 - 1) / (UT / 2) : 0;
  return it;
}

// Joins the states of an item's parts, in order, into st: part 0 at `first`, part w at later + w * stride. Two rows or
// fewer leave three quarters of a state's lanes without a row (four or fewer: half), which then take other parts.
template <int DH, int NT>
__device__ __forceinline__ void join_states(SoftState<DH, NT>& st, const float* first, const float* later, int stride,
                                            int parts, int R) {
  constexpr int ROWS = 8 * NT;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int fold = NT > 1 || R > 4 ? 1 : (R > 2 ? 2 : 4);  // parts side by side
  const int tc = t % (4 / fold), side = t / (4 / fold);    // column pair and side of this lane
  st.clear();
  constexpr int UN = DH / 16 * NT >= 8 ? 2 : 4;  // parts in flight (on each side)
  for (int w0 = 0; w0 < parts; w0 += UN * fold) {
    float4 ml[UN][NT], o[UN][NT][DH / 16];
#pragma unroll
    for (int y = 0; y < UN; ++y) {
      const int w = w0 + y * fold + side;
      const float* s = w == 0 ? first : later + (int64_t)w * stride;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        ml[y][nt] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
        const bool live = w < parts && nt * 8 + 2 * tc < R;
        if (live) ml[y][nt] = __ldcg(reinterpret_cast<const float4*>(s + ROWS * DH) + nt * 4 + tc);
#pragma unroll
        for (int x = 0; x < DH / 16; ++x) {
          o[y][nt][x] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (live) o[y][nt][x] = __ldcg(reinterpret_cast<const float4*>(s) + (x * NT + nt) * 32 + g * 4 + tc);
        }
      }
    }
    // a part that saw nothing, or nothing but NaN, has no maximum: its sums count as they are
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mn = st.m[nt][i];
#pragma unroll
        for (int y = 0; y < UN; ++y) mn = fmaxf(mn, i ? ml[y][nt].y : ml[y][nt].x);
        f[i] = st.m[nt][i] == -INFINITY ? 1.f : exp2_fast(st.m[nt][i] - mn);
        st.m[nt][i] = mn;
        st.l[nt][i] *= f[i];
      }
#pragma unroll
      for (int x = 0; x < DH / 16; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[x][nt][i] *= f[i & 1];
#pragma unroll
      for (int y = 0; y < UN; ++y) {
        const float f0 = ml[y][nt].x == -INFINITY ? 1.f : exp2_fast(ml[y][nt].x - st.m[nt][0]);
        const float f1 = ml[y][nt].y == -INFINITY ? 1.f : exp2_fast(ml[y][nt].y - st.m[nt][1]);
        st.l[nt][0] += ml[y][nt].z * f0;
        st.l[nt][1] += ml[y][nt].w * f1;
#pragma unroll
        for (int x = 0; x < DH / 16; ++x) {
          st.o[x][nt][0] += o[y][nt][x].x * f0;
          st.o[x][nt][1] += o[y][nt][x].y * f1;
          st.o[x][nt][2] += o[y][nt][x].z * f0;
          st.o[x][nt][3] += o[y][nt][x].w * f1;
        }
      }
    }
  }
  if (fold > 1)  // the sides meet
    for (int d = 4 / fold; d < 4; d <<= 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float om = __shfl_xor_sync(0xffffffffu, st.m[0][i], d), mn = fmaxf(st.m[0][i], om);
        const float f = st.m[0][i] == -INFINITY ? 1.f : exp2_fast(st.m[0][i] - mn);
        st.m[0][i] = mn;
        st.l[0][i] *= f;
        st.l[0][i] += __shfl_xor_sync(0xffffffffu, st.l[0][i], d);
#pragma unroll
        for (int x = 0; x < DH / 16; ++x)
#pragma unroll
          for (int j = i; j < 4; j += 2) {
            st.o[x][0][j] *= f;
            st.o[x][0][j] += __shfl_xor_sync(0xffffffffu, st.o[x][0][j], d);
          }
      }
    }
}

// The late join. What the warps of a CTA hold of one item at its end is joined in the CTA's
// shared memory first, so that an item shared by several CTAs has one state of each in the workspace, and one of the warp that
// holds its last unit. `first` and `last` are the warps that share the item, `wpc` warps to a CTA.
struct Join {
  int row0, n, h, first, last, wpc;
  int b, pos, odd;  // odd: the open page holds an infinity or NaN
  __device__ __forceinline__ int parts() const { return (last - 1) / wpc - first / wpc + 2; }
};

// Joins a tile (16 dims x of the 8 rows nt) of `parts` states, in order; get(part, i) is float4 i of a state. The code runs a
// few times on an SM at the end of a call, and fetching it costs as much as its loads and sums: a tile at a time keeps it
// small. No load is conditional (a branch around each kept them apart): a place without a part reads the last one and counts
// it 0 times, columns of no row come to nothing. A part that saw nothing, or nothing but NaN, has no maximum: its sums count
// as they are.
template <int DH, int NT, typename Get>
__device__ __forceinline__ void merge_tile(Get get, int parts, int x, int nt, float (&m)[2], float (&l)[2], float (&acc)[4]) {
  constexpr int UN = 4;
  const int lane = threadIdx.x & 31, t = lane & 3;
  m[0] = m[1] = -INFINITY;
  l[0] = l[1] = acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
#pragma unroll 1
  for (int w0 = 0; w0 < parts; w0 += UN) {
    float4 ml[UN], o[UN];
#pragma unroll
    for (int y = 0; y < UN; ++y) {
      const int w = min(w0 + y, parts - 1);
      ml[y] = get(w, 8 * NT * DH / 4 + nt * 4 + t);
      o[y] = get(w, (x * NT + nt) * 32 + lane);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float mn = m[i];
#pragma unroll
      for (int y = 0; y < UN; ++y) mn = fmaxf(mn, i ? ml[y].y : ml[y].x);
      const float f = m[i] == -INFINITY ? 1.f : exp2_fast(m[i] - mn);
      m[i] = mn;
      l[i] *= f;
      acc[i] *= f;
      acc[i + 2] *= f;
#pragma unroll
      for (int y = 0; y < UN; ++y) {
        const float my = i ? ml[y].y : ml[y].x;
        const float fy = w0 + y >= parts ? 0.f : (my == -INFINITY ? 1.f : exp2_fast(my - mn));
        l[i] += (i ? ml[y].w : ml[y].z) * fy;
        acc[i] += (i ? o[y].y : o[y].x) * fy;
        acc[i + 2] += (i ? o[y].w : o[y].z) * fy;
      }
    }
  }
}

// A tile of the states of `parts` warps, one after the other in shared memory `pitch` bytes apart, into one state.
template <int DH, int NT>
__device__ __noinline__ void gather_tile(const unsigned char* from, int pitch, int parts, int x, int nt, float* to) {
  const int lane = threadIdx.x & 31;
  float m[2], l[2], acc[4];
  merge_tile<DH, NT>([&](int w, int i) { return reinterpret_cast<const float4*>(from + w * pitch)[i]; }, parts, x, nt, m, l, acc);
  __stcg(reinterpret_cast<float4*>(to) + (x * NT + nt) * 32 + lane, make_float4(acc[0], acc[1], acc[2], acc[3]));
  if (x == 0 && lane < 4) __stcg(reinterpret_cast<float4*>(to + 8 * NT * DH) + nt * 4 + lane, make_float4(m[0], m[1], l[0], l[1]));
}

// A tile of an item whose states are all in the workspace, to the output. states: of the warps that hold last units; groups:
// of CTAs, each in the place of its first warp of the item. out, lse: of the item's first row and head. (By value: a reference
// to the kernel's parameters put them into local memory, a miss away: a join took 6 us against 4.)
template <typename T, int DH, int NT>
__device__ __noinline__ void join_tile(const Join* join, const float* states, const float* groups, int x, int nt, int group,
                                       T* out, int64_t o_sr, int64_t o_sh, float* lse, int Hq, void* tail, int Hkv, int P,
                                       int window) {
  using SH = SplitShape<DH, NT>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Join j = *join;
  const int R = j.n * group, parts = j.parts(), cta0 = j.first / j.wpc;
  float m[2], l[2], acc[4];
  merge_tile<DH, NT>(
      [&](int w, int i) {
        const float* s = w == parts - 1 ? states + (int64_t)j.last * SH::STATE
                                        : groups + (int64_t)max(j.first, (cta0 + w) * j.wpc) * SH::STATE;
        return __ldcg(reinterpret_cast<const float4*>(s) + i);
      },
      parts, x, nt, m, l, acc);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int rr = nt * 8 + 2 * t + i;
    if (rr >= R) continue;
    const int q = rr / group, gq = rr - q * group;
    T* o = out + q * o_sr + gq * o_sh + x * 16 + g;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    o[0] = from_f32<T>(acc[i] * inv);
    o[8] = from_f32<T>(acc[i + 2] * inv);
    if (lse && g == 0 && x == 0)
      lse[(int64_t)q * Hq + gq] = l[i] == 0.f ? -INFINITY : (m[i] - ATTN_SHIFT + log2f(l[i])) * 0.69314718055994531f;
  }
  if (__builtin_expect(j.odd != 0, 0)) {
    __syncwarp();
    const int n_full = (j.pos + j.n) / P;
    const PagedCache c{nullptr, tail, nullptr, 0, 0, 0, Hkv, P};
    for (int rr = nt * 8; rr < min(R, nt * 8 + 8); ++rr) {
      const int q = rr / group, qp = j.pos + q;
      add_odd<T, DH>(open_values<T, DH>(c, j.b, j.h, n_full), n_full * P, window > 0 ? qp - window + 1 : 0, qp + 1, x * 16 + lane,
                     x * 16 + 16, 32, out + q * o_sr + (rr - q * group) * o_sh);
    }
  }
}

template <typename T, int DH, int NT, bool LATE, bool PROBE = false>
__global__ void __launch_bounds__(SplitShape<DH, NT>::WARPS * 32, 1)
    paged_split_kernel(AttnParams p, int32_t* counters, float* states) {
  using SH = SplitShape<DH, NT>;
  constexpr int WARPS = SH::WARPS, NS = SH::NS, ROWS = 8 * NT, UT = SH::UT, TT = SH::TT;
  constexpr int TG = NT >= 3 ? 2 : UT / 16;  // 64 tokens' scores beside 24 or 32 rows' numerators do not fit the registers
  extern __shared__ __align__(128) unsigned char split_smem[];
  __shared__ int warp_sums[WARPS];
  // late joins: the item that each warp leaves unfinished (-1: none), and items whose last part is this CTA's
  __shared__ int held[WARPS];
  __shared__ Join held_join[WARPS], joins[2 * WARPS];
  __shared__ int n_joins;
  unsigned char* ring = split_smem;
  uint64_t* bars = reinterpret_cast<uint64_t*>(split_smem + SH::RING);
  int* s_first = reinterpret_cast<int*>(split_smem + SH::RING + SH::BAR_BYTES);  // first unit of sequence b (B + 1)
  int* s_row = s_first + p.B + 1;
  int* s_pos = s_row + p.B + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int P = p.c.P, lp = 31 - __clz(P), Hkv = p.c.Hkv, group = p.Hq / Hkv;
  const int rec = 2 * P * DH + 16;
  // a unit in shared memory: records of Pe tokens (whole ones, or a part of one with its scales)
  const int Pe = min(P, UT), lpe = 31 - __clz(Pe), per = UT >> lpe, rec_e = 2 * Pe * DH + 16;
  uint64_t* bar = bars + warp * NS;
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(bar + i, 1);
    fence_mbar_init();
  }
  if (tid == 0) n_joins = 0;
  if (tid < WARPS) held[tid] = -1;
  pdl_wait();
  pdl_launch_dependents();
  // where each sequence's units begin
  {
    const int chunk = (p.B + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = min(p.B, tid * chunk), b1 = min(p.B, b0 + chunk);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      const int r0 = p.start[b], n = p.start[b + 1] - r0, ps = p.pos[b];
      int units = 0;
      if (r0 < 0 || n < 0 || r0 + n > p.n_rows || n > p.max_new)
        record_error(DEV_INDEX_RANGE, K_PAGED_ATTN, b, n);
      else if (ps < 0 || (int64_t)ps + n > (int64_t)p.c.max_pages * P + (P - 1))
        record_error(DEV_POS_RANGE, K_PAGED_ATTN, b, ps);
      else
        units = n > 0 ? (item_of<UT>(r0, n, ps, lp, p.window).units + SPLIT_ITEM_COST) * Hkv : 0;
      s_first[b + 1] = units;
      s_row[b] = r0;
      s_pos[b] = ps;
      if (b == p.B - 1) s_row[b + 1] = r0 + n;
      sum += units;
    }
    int inc = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int at = inc - sum;
    for (int w = 0; w < warp; ++w) at += warp_sums[w];
    for (int b = b0; b < b1; ++b) {
      at += s_first[b + 1];
      s_first[b + 1] = at;
    }
    if (tid == 0) s_first[0] = 0;
    __syncthreads();
  }
  const int total = s_first[p.B];
  if (total == 0) return;
  const int n_work = min((int)gridDim.x * WARPS, (total + SPLIT_MIN_UNITS - 1) / SPLIT_MIN_UNITS);
  // neighbours share an SM (which spreads the joins over the SMs), as few to each as leaves none without
  const int wpc = (n_work + gridDim.x - 1) / gridDim.x;
  const int me = warp < wpc ? blockIdx.x * wpc + warp : n_work;
  // even shares, the first `over` warps with one more (32-bit divisions only)
  const int share = total / n_work, over = total % n_work;
  auto first_of = [&](int w) { return w * share + min(w, over); };
  auto owner_of = [&](int u) { return u < (share + 1) * over ? u / (share + 1) : over + (u - (share + 1) * over) / share; };
  const int u0 = me < n_work ? first_of(me) : 0, u1 = me < n_work ? first_of(me + 1) : 0;
  const int32_t* table = p.c.table;

  // A run of units of one item: [k, end) of it. Places in the order of all items count SPLIT_ITEM_COST empty ones before an
  // item's units.
  struct Run {
    Item it;
    int b, h, k, end;
    int at;    // place of the item's first unit
    int next;  // place after the run
  };
  // the first run from place u on; false when only empty places are left
  auto open = [&](Run& r, int u) {
    while (u < u1) {
      int lo = 0, hi = p.B - 1;
      while (lo < hi) {  // the last sequence that begins at or before u
        const int mid = (lo + hi + 1) / 2;
        if (s_first[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      r.b = lo;
      r.it = item_of<UT>(s_row[lo], s_row[lo + 1] - s_row[lo], s_pos[lo], lp, p.window);
      const int size = r.it.units + SPLIT_ITEM_COST, in = u - s_first[lo];
      r.h = in / size;
      r.at = u - in % size + SPLIT_ITEM_COST;
      r.k = max(0, u - r.at);
      r.end = min(r.it.units, u1 - r.at);
      r.next = min(u1, r.at + r.it.units);
      if (r.k < r.end) return true;
      u = r.next;
    }
    return false;
  };

  // ---- copies: `ahead` runs NS units before the one at work. Records are read once: they leave the L2 first, so that they
  // push out neither the states nor the code that runs once at the end (64 sequences 65 -> 61 us).
  const uint64_t once = l2_policy_evict_first();
  Run ahead{};
  bool more = true;     // it has a unit to copy
  int batch = 0;        // page of the item that lane 0's table entry stands for
  int entry = 0, entry_next = 0;
  auto load_entry = [&](int page) {
    return page < ahead.it.p1 ? table[ahead.b * p.c.table_sb + page] : 0;
  };
  auto begin_ahead = [&](int u) {
    more = open(ahead, u);
    if (!more) return;
    batch = ahead.it.p0 + ((ahead.k * UT) >> lp);
    entry = load_entry(batch + lane);
    entry_next = load_entry(batch + 32 + lane);
  };
  bool skip = PROBE && me == p.probe;
  auto issue = [&](int slot) {
    if constexpr (PROBE) {
      if (skip) {  // a copy that never comes
        skip = false;
        if (++ahead.k == ahead.end) begin_ahead(ahead.next);
        return;
      }
    }
    unsigned char* dst = ring + (warp * NS + slot) * SH::STAGE;
    if (ahead.k < ahead.it.nu8) {
      const int page = ahead.it.p0 + ((ahead.k * UT) >> lp);
      if (page >= batch + 32) {
        batch += 32;
        entry = entry_next;
        entry_next = load_entry(batch + 32 + lane);
      }
      // a unit's pages beyond the last full one are copies of it (masked, but finite)
      const int at = min(page + (lane < per ? lane : 0), ahead.it.p1 - 1) - batch;
      const unsigned char* src = record_of(p.c, __shfl_sync(0xffffffffu, entry, at), ahead.h, rec, ahead.b);
      if (lane == 0) mbar_arrive_expect_tx(bar + slot, (uint32_t)(per * rec_e));
      __syncwarp();
      if (P <= UT) {
        if (lane < per) bulk_g2s_hint(dst + lane * rec_e, src, (uint32_t)rec_e, bar + slot, once);
      } else if (lane < 3) {  // keys, values and scales of a part of the page
        const int in = (ahead.k * UT) & (P - 1);
        bulk_g2s_hint(dst + lane * UT * DH, src + lane * P * DH + (lane < 2 ? in * DH : 0), lane < 2 ? UT * DH : 16, bar + slot,
                      once);
      }
    } else if (lane == 0) {
      const int t0 = (ahead.k - ahead.it.nu8) * TT;  // token of the open page
      const int left = min(ahead.it.len - (ahead.it.p1 << lp) - t0, TT);
      const uint32_t bytes = (uint32_t)((left + 15) >> 4) * 16 * DH * 2;
      const T* src = reinterpret_cast<const T*>(p.c.tail) +
                     ((((int64_t)ahead.b * Hkv + ahead.h) * 2 + (ahead.it.p1 & 1)) * 2) * ((int64_t)P * DH) + t0 * DH;
      mbar_arrive_expect_tx(bar + slot, 2 * bytes);
      bulk_g2s(dst, src, bytes, bar + slot);
      bulk_g2s(dst + UT * DH, src + (int64_t)P * DH, bytes, bar + slot);
    }
    __syncwarp();
    if (++ahead.k == ahead.end) begin_ahead(ahead.next);
  };

  RowTile<T, DH, NT> rt;
  SoftState<DH, NT> st;
  Run run;
  typename RowTile<T, DH, NT>::Raw raw;
  begin_ahead(u0);
  const bool idle = !more;
  run = ahead;
  // the first run's queries are fetched before the copies fill the memory's queues
  if (!idle) rt.fetch(p, run.it.row0, run.h, group, 0, run.it.n * group, raw);
  int issued = 0;
  for (; issued < NS && more; ++issued) issue(issued);
  bool ok = true;
  int step = 0;  // units consumed
  for (bool first = true; !idle && (first || open(run, run.next)); first = false) {
    if (!first) rt.fetch(p, run.it.row0, run.h, group, 0, run.it.n * group, raw);
    rt.finish(p, run.it.pos, group, 0, run.it.n * group, raw);
    const Item& it = run.it;
    const int R = it.n * group;
    st.clear(ok ? 0.f : NAN);
    const int qhi = it.pos + it.n - 1;
    uint32_t odd = 0u;  // the open page holds an infinity or NaN
    const int last = ok ? run.end : run.k;
    for (int k = run.k; k < last; ++k, ++step) {
      const int slot = step % NS;
      const unsigned char* src = ring + (warp * NS + slot) * SH::STAGE;
      if (!mbar_wait_bounded(bar + slot, (step / NS) & 1, K_PAGED_ATTN, 1)) {
        // This run and the warp's later ones are NaN; they arrive all the same, so that the others' counters come back to zero.
        ok = false;
        st.clear(NAN);
        break;  // (step stays)
      }
      if (k < it.nu8) {
        const int tok0 = (it.p0 << lp) + k * UT, limit = it.p1 << lp;
        const bool mask = tok0 + UT - 1 > min(it.pos, limit - 1) || (p.window > 0 && tok0 <= qhi - p.window);
#pragma unroll 1
        for (int y = 0; y < UT / 16; y += TG) {  // 16-token groups at a time
          const unsigned char *kp[TG], *vp[TG];
          float ks[TG], lv[TG], iv[TG];
#pragma unroll
          for (int x = 0; x < TG; ++x) {
            const unsigned char* rp = src + (((y + x) * 16) >> lpe) * rec_e;
            kp[x] = rp + (((y + x) * 16) & (Pe - 1)) * DH;
            vp[x] = kp[x] + Pe * DH;
            const float4 sc = *reinterpret_cast<const float4*>(rp + 2 * Pe * DH);
            ks[x] = sc.x;
            value_factors(sc, lv[x], iv[x]);
          }
          attend_codes<T, DH, NT, TG>(rt, st, kp, vp, ks, lv, iv, tok0 + y * 16, limit, p.window, mask);
        }
      } else {
        const int tok0 = (it.p1 << lp) + (k - it.nu8) * TT;
        unsigned char* v = ring + (warp * NS + slot) * SH::STAGE + UT * DH;
        if (clean_values<T>(v, (min(it.len - tok0, TT) + 15) / 16 * 2 * DH)) odd = 1u;
        attend_tail<T, DH, NT, TT / 16, true>(rt, st, reinterpret_cast<const T*>(src), reinterpret_cast<const T*>(v), tok0,
                                              it.len, p.window, odd);
      }
      __syncwarp();  // every lane has read the unit
      if (more) {
        issue(slot);
        ++issued;
      }
    }
    // ---- the run's end: out, or into the workspace
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float& l = st.l[nt][i];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
      }
    bool write = run.k == 0 && run.end == it.units;
    if (!write) {
      const int wa = owner_of(run.at), wb = owner_of(run.at + it.units - 1), item = run.b * Hkv + run.h;
      Join join{it.row0, it.n, run.h, wa, wb, wpc, run.b, it.pos, (int)odd};
      if (LATE && run.end < it.units) {
        // (the warp's last run) stays in the registers until the CTA's warps are done
        if (lane == 0) {
          held[warp] = item;
          held_join[warp] = join;
        }
        break;
      }
      // late joins: one a warp; others: the first of an item that others began, the second of one that it begins
      float* mine = states + (LATE ? (int64_t)me : (int64_t)me * 2 + (run.k > 0 ? 0 : 1)) * SH::STATE;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (nt * 8 + 2 * t >= R) continue;  // columns of no row are not written, and come to nothing where they are read
#pragma unroll
        for (int x = 0; x < DH / 16; ++x)
          __stcg(reinterpret_cast<float4*>(mine) + (x * NT + nt) * 32 + lane,
                 make_float4(st.o[x][nt][0], st.o[x][nt][1], st.o[x][nt][2], st.o[x][nt][3]));
        if (g == 0)
          __stcg(reinterpret_cast<float4*>(mine + ROWS * DH) + nt * 4 + t,
                 make_float4(st.m[nt][0], st.m[nt][1], st.l[nt][0], st.l[nt][1]));
      }
      __threadfence();
      __syncwarp();
      int32_t* cnt = counters + item;
      int before = 0;
      if (lane == 0) before = atomicAdd(cnt, 1 + ((int)odd << 16));  // arrivals, and above them those of odd parts
      before = __shfl_sync(0xffffffffu, before, 0);
      if ((before & 0xffff) == (LATE ? join.parts() - 1 : wb - wa)) {
        __threadfence();
        if (lane == 0) *cnt = 0;
        odd |= before >> 16;
        join.odd = odd;
        if constexpr (LATE) {
          if (lane == 0) joins[atomicAdd(&n_joins, 1)] = join;
        } else {
          const float* later = states + (int64_t)wa * 2 * SH::STATE;
          join_states<DH, NT>(st, later + SH::STATE, later, 2 * SH::STATE, wb - wa + 1, R);
          write = true;
        }
      }
    }
    if (write) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int rr = nt * 8 + 2 * t + i;
          if (rr >= R) continue;
          const float l = st.l[nt][i], inv = l == 0.f ? 0.f : 1.f / l;
          const int64_t row = it.row0 + rr / group;
          const int hq = run.h * group + rr % group;
          T* o = reinterpret_cast<T*>(p.out) + row * p.o_sr + (int64_t)hq * p.o_sh;
#pragma unroll
          for (int x = 0; x < DH / 16; ++x) {
            o[x * 16 + g] = from_f32<T>(l == 0.f ? 0.f : st.o[x][nt][i] * inv);
            o[x * 16 + 8 + g] = from_f32<T>(l == 0.f ? 0.f : st.o[x][nt][i + 2] * inv);
          }
          if (p.lse && g == 0)
            p.lse[row * p.Hq + hq] = l == 0.f ? -INFINITY : (st.m[nt][i] - ATTN_SHIFT + log2f(l)) * 0.69314718055994531f;
        }
      if (__builtin_expect(odd != 0u, 0)) {
        __syncwarp();
        const T* tv = open_values<T, DH>(p.c, run.b, run.h, it.p1);
#pragma unroll 1
        for (int rr = 0; rr < R; ++rr) {
          const int q = rr / group, qp = it.pos + q;
          add_odd<T, DH>(tv, it.p1 << lp, p.window > 0 ? qp - p.window + 1 : 0, qp + 1, lane, DH, 32,
                         reinterpret_cast<T*>(p.out) + (it.row0 + q) * p.o_sr + (int64_t)(run.h * group + rr % group) * p.o_sh);
        }
      }
    }
  }
  if (!ok)  // no copy of this warp may still be in flight when its CTA ends
    for (int i = step + 1; i < issued; ++i) mbar_wait_bounded(bar + i % NS, (i / NS) & 1, K_PAGED_ATTN, 2);
  if constexpr (LATE) {
    // What the CTA's warps leave unfinished, joined by all of them in the rings, which are done with: one state a CTA and
    // item goes to the workspace, and the last to come joins an item's. (12 parts of 20 rows of head dim 128: one warp alone
    // took 16 to 20 us, all warps of a CTA over 12 states in the workspace 9; this way 4 us here and 4 for each join.)
    __syncthreads();
    constexpr int PITCH = NS * SH::STAGE;
    static_assert(SH::STATE * 4 <= PITCH, "a warp's state fits its ring");
    if (held[warp] >= 0) {
      float4* mine = reinterpret_cast<float4*>(ring + warp * PITCH);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 0; x < DH / 16; ++x)
          mine[(x * NT + nt) * 32 + lane] = make_float4(st.o[x][nt][0], st.o[x][nt][1], st.o[x][nt][2], st.o[x][nt][3]);
        if (g == 0) mine[ROWS * DH / 4 + nt * 4 + t] = make_float4(st.m[nt][0], st.m[nt][1], st.l[nt][0], st.l[nt][1]);
      }
    }
    __syncthreads();
    float* groups = states + (int64_t)gridDim.x * WARPS * SH::STATE;
    auto leads = [&](int w) { return held[w] >= 0 && (w == 0 || held[w - 1] != held[w]); };
    int task = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (!leads(w)) continue;
      int count = 1;
      while (w + count < WARPS && held[w + count] == held[w]) ++count;
      for (int i = 0; i < NT * (DH / 16); ++i, ++task)
        if (task % WARPS == warp)
          gather_tile<DH, NT>(ring + w * PITCH, PITCH, count, i / NT, i % NT, groups + (int64_t)(blockIdx.x * wpc + w) * SH::STATE);
    }
    __threadfence();
    __syncthreads();
    if (lane == 0 && leads(warp)) {
      int32_t* cnt = counters + held[warp];
      Join join = held_join[warp];
      for (int w = warp + 1; w < WARPS && held[w] == held[warp]; ++w) join.odd |= held_join[w].odd;
      const int before = atomicAdd(cnt, 1 + (join.odd << 16));
      if ((before & 0xffff) == join.parts() - 1) {
        *cnt = 0;
        join.odd |= before >> 16;
        joins[atomicAdd(&n_joins, 1)] = join;
      }
      __threadfence();
    }
    __syncthreads();
    constexpr int TILES = NT * (DH / 16);
    for (int i = warp; i < n_joins * TILES; i += WARPS) {
      const Join* j = joins + i / TILES;
      const int64_t row = j->row0;
      const int hq = j->h * group;
      join_tile<T, DH, NT>(j, states, groups, i % TILES / NT, i % NT, group,
                           reinterpret_cast<T*>(p.out) + row * p.o_sr + (int64_t)hq * p.o_sh, p.o_sr, p.o_sh,
                           p.lse ? p.lse + row * p.Hq + hq : nullptr, p.Hq, p.c.tail, Hkv, P, p.window);
    }
  }
}

}  // namespace ta
