// Low-rank adapters of many requests beside a shared projection, forward and backward.
//   t = s_a x A_a^T,  out = y + t B_a^T                      on the rows of each sequence, a = which[sequence]
//   u = s_a dy B_a,   dx = u A_a,  dA_a = u^T x,  dB_a = dy^T t   (sums over the rows of all sequences with adapter a)
// A rank of 8 to 128 gives each element of x and y 2 r operations for its 2 bytes: below the 250 an element that the memory allows the
// tensor cores, so the kernels are bound by the rows' bytes (by latency where there are few rows). That is why they use the
// warp-level matrix instruction, whose fragments come from rows of any length.
// Few rows of a sequence (decoding) take one kernel for both products; many take two, t going by way of memory (64 bytes a row at rank
// 16): its columns and the output's are then shared out over the GPU apart, and no CTA waits for another but to sum t.
// t is held in fp32 and enters its product as two 16-bit numbers, high and low: 16 bits of it (22 in f16), so that the output's one
// rounding is what is seen.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace ta {

struct AdapterParams {
  const void *x, *y;  // rows (n, K) and (n, N); y null: 0
  void* out;          // (n, N), may be y
  int64_t x_sr, y_sr, o_sr;
  const void *u, *v;  // the adapters' factors: u contracts K, v gives N. Forward (n_adapters, r, K) and (n_adapters, N, r); TRANS
                      // (n_adapters, K, r) and (n_adapters, r, N)
  const float* scale; // (n_adapters,) or null (1)
  const int32_t *start, *which;
  int n_rows, B, K, N, r, n_adapters;
  int tiles;          // of a sequence that the grid has clusters (or CTAs) for
  void* t;            // (2, n, r): t's high and low parts, or null (one kernel for both products, nothing kept)
  float* t_by;        // (n,), f16: what a row of t is to be multiplied by
};

constexpr int ADAPTER_THREADS = 256;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {  // zeros where there is nothing to read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void stsm4(uint32_t a, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T> __device__ __forceinline__ float2 widen2(uint32_t x);
template <> __device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 widen2<__half>(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
template <typename T> __device__ __forceinline__ uint32_t narrow2(float a, float b);
template <> __device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t narrow2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The B operand's 16 x 16 block (k k0.., n n0..), from n-major rows (k contiguous) or, TR, from k-major ones. pitch in bytes.
template <bool TR>
__device__ __forceinline__ void load_b(uint32_t (&b)[4], uint32_t base, int pitch, int n0, int k0, int lane) {
  if (TR)
    ldsm4t(b, base + (k0 + (lane & 15)) * pitch + (n0 + (lane >> 4) * 8) * 2);
  else
    ldsm4(b, base + (n0 + (lane >> 4) * 8 + (lane & 7)) * pitch + (k0 + ((lane >> 3) & 1) * 8) * 2);
}

template <int TM, int RP, bool TRANS, bool FUSED>
struct AdapterShape {
  static constexpr int WM = TM / 16, WK = 8 / WM;              // warps by rows, and by columns
  static constexpr int KC = TM == 16 || RP <= 32 ? 128 : 64;   // columns of x, and of the output, in a stage: 256 bytes of a row where
                                                               // they fit (of 128 the memory gives two thirds as much a second)
  static constexpr int STAGES = KC == 128 ? 3 : 4;
  static constexpr int XP = KC * 2 + 16, RPP = RP * 2 + 16;    // pitches of rows by columns and by rank
  static constexpr int F = TRANS ? KC * RPP : RP * XP;         // a stage's part of u, ...
  static constexpr int G = !FUSED ? 0 : TRANS ? RP * XP : KC * RPP;  // ... and of v
  static constexpr int STAGE = TM * XP + (F > G ? F : G);
  static constexpr int PART = WK * TM * RP * 4;
  static constexpr int BYTES = STAGES * STAGE + PART + (FUSED ? 2 * TM * RPP + TM * 4 : 0);
};

// The output's 16 x 8 NT block of a warp, from y's tile at `tile` (pitch XP): t's rows times v, added, rounded once and written back there;
// whole 16-byte pieces then leave for rows below `rows` and columns below `cols` of `out` (the CTA's corner).
template <typename T, int RP, int NT, bool TRANS>
__device__ __forceinline__ void add_product(unsigned char* tile, int xp, uint32_t vs, int vp, uint32_t hi, uint32_t lo, int tp, const float* row_by,
                                            bool with_y, int m0, int n0, int lane, T* out, int64_t o_sr, int rows, int cols) {
  constexpr bool FROM_Y = !std::is_same<T, __half>::value;  // the sum begins with y (f16's rows have a factor of their own)
  const uint32_t y_at = smem_u32(tile) + (m0 + (lane & 15)) * xp + (n0 + (lane >> 4) * 8) * 2;
  const uint32_t t_at = (m0 + (lane & 15)) * tp + (lane >> 4) * 16;
  float o[NT][4];
  auto begin = [&](auto set) {
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t y[4] = {0u, 0u, 0u, 0u};
      if (with_y) ldsm4(y, y_at + n * 16);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float2 f = widen2<T>(y[h]);
        set(o[n + h / 2][h % 2 * 2], f.x, h % 2);
        set(o[n + h / 2][h % 2 * 2 + 1], f.y, h % 2);
      }
    }
  };
  if (FROM_Y) {
    begin([](float& a, float y, int) { a = y; });
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  }
#pragma unroll
  for (int kk = 0; kk < RP / 16; ++kk) {
    uint32_t th[4], tl[4];
    ldsm4(th, hi + t_at + kk * 32);
    ldsm4(tl, lo + t_at + kk * 32);
#pragma unroll
    for (int n = 0; n < NT / 2; ++n) {
      uint32_t vb[4];
      load_b<TRANS>(vb, vs, vp, n0 + n * 16, kk * 16, lane);
      mma16<T>(o[2 * n], th, vb[0], vb[1]);
      mma16<T>(o[2 * n + 1], th, vb[2], vb[3]);
      mma16<T>(o[2 * n], tl, vb[0], vb[1]);
      mma16<T>(o[2 * n + 1], tl, vb[2], vb[3]);
    }
  }
  if (!FROM_Y) {
    const float by[2] = {row_by[m0 + lane / 4], row_by[m0 + lane / 4 + 8]};
    begin([&](float& a, float y, int h) { a = fmaf(a, by[h], y); });
  }
#pragma unroll
  for (int n = 0; n < NT; n += 2) {
    const uint32_t r4[4] = {narrow2<T>(o[n][0], o[n][1]), narrow2<T>(o[n][2], o[n][3]), narrow2<T>(o[n + 1][0], o[n + 1][1]),
                            narrow2<T>(o[n + 1][2], o[n + 1][3])};
    stsm4(y_at + n * 16, r4);
  }
  __syncwarp();
  constexpr int STEP = 32 / NT;
  const int m = m0 + lane / NT, c = n0 + lane % NT * 8;
  if (c < cols) {
#pragma unroll
    for (int q = 0; q < NT / 2; ++q)
      if (m + q * STEP < rows)
        *reinterpret_cast<uint4*>(out + (m + q * STEP) * o_sr + c) = *reinterpret_cast<const uint4*>(tile + (m + q * STEP) * xp + c * 2);
  }
}

// A cluster of CTAs takes a tile of a sequence's rows. Each contracts a share of x's columns; the partial t meet through distributed
// shared memory, summed in the ranks' order.
// FUSED (tiles of 16 rows): each CTA sums t for itself and adds its share of the output's columns. The stages of both halves go through one
// ring of asynchronous copies, so that the second half's first stages arrive while t is summed.
// Otherwise (tiles of 64) each CTA sums and writes a share of t's rows.
template <typename T, int TM, int RP, bool TRANS, bool FUSED>
__global__ void __launch_bounds__(ADAPTER_THREADS, RP <= 32 ? (FUSED ? 4 : 3) : RP == 64 ? 2 : 1)
    adapter_kernel(const __grid_constant__ AdapterParams p) {
  using S = AdapterShape<TM, RP, TRANS, FUSED>;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const ring = smem;
  float* const part = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE);
  unsigned char* const hi = smem + S::STAGES * S::STAGE + S::PART;
  unsigned char* const lo = hi + TM * S::RPP;
  float* const row_by = reinterpret_cast<float*>(lo + TM * S::RPP);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int tile0 = blockIdx.x / cs, b = blockIdx.y;
  const T* const X = reinterpret_cast<const T*>(p.x);
  const T* const Y = reinterpret_cast<const T*>(p.y);
  T* const O = reinterpret_cast<T*>(p.out);
  pdl_wait();
  pdl_launch_dependents();

  // rows [r0, r1) as they are (y, or 0), or NaN
  auto plain = [&](int r0, int r1, bool nan) {
    if (!FUSED || (p.out == p.y && !nan)) return;
    const int pieces = p.N / 8;
    for (int64_t i = (int64_t)blockIdx.x * ADAPTER_THREADS + tid; i < (int64_t)(r1 - r0) * pieces;
         i += (int64_t)gridDim.x * ADAPTER_THREADS) {
      const int64_t row = r0 + i / pieces;
      const int c = (int)(i % pieces) * 8;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (nan) v = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      else if (Y) v = *reinterpret_cast<const uint4*>(Y + row * p.y_sr + c);
      *reinterpret_cast<uint4*>(O + row * p.o_sr + c) = v;
    }
  };
  auto bound = [&](int r) { return min(max(r, 0), p.n_rows); };
  if (b == p.B) {  // rows of no sequence
    plain(0, bound(p.start[0]), false);
    plain(bound(p.start[p.B]), p.n_rows, false);
    return;
  }
  const int r0 = bound(p.start[b]), r1 = bound(p.start[b + 1]);
  const int a = p.which[b];
  if (a < 0 || a >= p.n_adapters) {
    if (a != -1 && blockIdx.x == 0 && tid == 0) record_error(DEV_INDEX_RANGE, K_ADAPTER, b, a);
    plain(r0, r1, a != -1);
    return;
  }
  const T* const U = reinterpret_cast<const T*>(p.u) + (int64_t)a * p.r * p.K;
  const T* const V = reinterpret_cast<const T*>(p.v) + (int64_t)a * p.r * p.N;
  const float scale = p.scale ? p.scale[a] : 1.f;
  const int wm = warp % S::WM, wk = warp / S::WM;
  const int kc = (p.K + S::KC - 1) / S::KC, nc = (p.N + S::KC - 1) / S::KC;
  const int k_first = kc * rank / cs, nk = kc * (rank + 1) / cs - k_first;
  const int n_first = nc * rank / cs, nn = FUSED ? nc * (rank + 1) / cs - n_first : 0;
  const uint32_t ring_at = smem_u32(ring), hi_at = smem_u32(hi), lo_at = smem_u32(lo);
  // a thread's pieces of a stage: of the rows, by columns; of a factor by rank (columns contiguous: u forward, v TRANS) or by column
  constexpr int CH = S::KC / 8, RH = RP / 8, RI = ADAPTER_THREADS / CH, CI = ADAPTER_THREADS / RH;
  const int pm = tid / CH, pc = tid % CH * 8, qm = tid / RH, qc = tid % RH * 8;
  const uint32_t row_to = ring_at + pm * S::XP + pc * 2, col_to = ring_at + TM * S::XP + qm * S::RPP + qc * 2;
  const bool whole_rank = p.r == RP;

  for (int row0 = r0 + tile0 * TM; row0 < r1; row0 += p.tiles * TM) {
    const int rows = min(TM, r1 - row0);
    const int mine = (rows - pm + RI - 1) / RI;  // this thread's rows: pm, pm + RI, ... (the others' places keep what they hold)
    const T* const x_at = X + (int64_t)(row0 + pm) * p.x_sr + pc;
    const T* const y_at = Y ? Y + (int64_t)(row0 + pm) * p.y_sr + pc : nullptr;
    auto issue = [&](int i) {
      if (i < nk + nn) {
        const bool first = i < nk;
        const uint32_t stage = (i % S::STAGES) * S::STAGE;
        const int c0 = (first ? k_first + i : n_first + i - nk) * S::KC, C = first ? p.K : p.N;
        const bool cut = c0 + S::KC > C;  // the columns end in this stage: u's and x's are filled up with zeros, y's do not matter
        const T* const from = (first ? x_at : y_at) + c0;
        const int64_t sr = first ? p.x_sr : p.y_sr;
        if (first || Y) {
          if (!cut) {
#pragma unroll
            for (int q = 0; q < TM / RI; ++q)
              if (q < mine) cp16(row_to + stage + q * RI * S::XP, from + q * RI * sr);
          } else {
            const bool real = c0 + pc < C;
#pragma unroll
            for (int q = 0; q < TM / RI; ++q)
              if (q < mine) cp16(row_to + stage + q * RI * S::XP, real ? from + q * RI * sr : X, real);
          }
        }
        const T* const W = first ? U : V;
        if (first != TRANS) {
          const T* const w = W + (int64_t)pm * C + c0 + pc;
          if (!cut && whole_rank) {
#pragma unroll
            for (int q = 0; q < (RP + RI - 1) / RI; ++q)
              if (RP % RI == 0 || pm + q * RI < RP) cp16(row_to + TM * S::XP + stage + q * RI * S::XP, w + (int64_t)q * RI * C);
          } else {
            for (int q = 0; q < (RP + RI - 1) / RI; ++q) {
              const int m = pm + q * RI;
              const bool real = m < p.r && c0 + pc < C;
              if (m < RP) cp16(row_to + TM * S::XP + stage + q * RI * S::XP, real ? w + (int64_t)q * RI * C : W, real);
            }
          }
        } else {
          const T* const w = W + (int64_t)(c0 + qm) * p.r + qc;
          if (!cut && whole_rank) {
#pragma unroll
            for (int q = 0; q < (S::KC + CI - 1) / CI; ++q)
              if (S::KC % CI == 0 || qm + q * CI < S::KC) cp16(col_to + stage + q * CI * S::RPP, w + q * CI * RP);
          } else {
            for (int q = 0; q < (S::KC + CI - 1) / CI; ++q) {
              const bool real = qc < p.r && c0 + qm + q * CI < C;
              if (qm + q * CI < S::KC) cp16(col_to + stage + q * CI * S::RPP, real ? w + (int64_t)q * CI * p.r : W, real);
            }
          }
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) issue(i);

    float acc[RP / 8][4];
#pragma unroll
    for (int n = 0; n < RP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    for (int i = 0; i < nk; ++i) {
      cp_wait<S::STAGES - 2>();
      __syncthreads();
      issue(i + S::STAGES - 1);
      const uint32_t xs = ring_at + (i % S::STAGES) * S::STAGE, us = xs + TM * S::XP;
#pragma unroll
      for (int kk = 0; kk < S::KC / 16 / S::WK; ++kk) {
        const int k0 = (kk * S::WK + wk) * 16;
        uint32_t xa[4];
        ldsm4(xa, xs + (wm * 16 + (lane & 15)) * S::XP + (k0 + (lane >> 4) * 8) * 2);
#pragma unroll
        for (int n = 0; n < RP / 16; ++n) {
          uint32_t ub[4];
          load_b<TRANS>(ub, us, TRANS ? S::RPP : S::XP, n * 16, k0, lane);
          mma16<T>(acc[2 * n], xa, ub[0], ub[1]);
          mma16<T>(acc[2 * n + 1], xa, ub[2], ub[3]);
        }
      }
    }
    // the warps' parts, the CTA's, the cluster's
    {
      float* const to = part + wk * TM * RP;
      const int m = wm * 16 + lane / 4, c = (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < RP / 8; ++n) {
        *reinterpret_cast<float2*>(to + m * RP + n * 8 + c) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(to + (m + 8) * RP + n * 8 + c) = make_float2(acc[n][2], acc[n][3]);
      }
    }
    __syncthreads();
    if (S::WK > 1) {
      for (int i = tid; i < TM * RP; i += ADAPTER_THREADS) {
        float s = part[i];
#pragma unroll
        for (int w = 1; w < S::WK; ++w) s += part[w * TM * RP + i];
        part[i] = s;
      }
    }
    if (cs > 1)
      cluster_sync_all();
    else
      __syncthreads();
    // a warp a row: t summed over the cluster, scaled, split into high and low parts
    for (int m = FUSED ? warp : warp * cs + rank; m < TM; m += ADAPTER_THREADS / 32 * (FUSED ? 1 : cs)) {
      constexpr int VL = (RP + 31) / 32;
      float s[VL];
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int c = lane + 32 * j;
        s[j] = 0.f;
        if (c < RP) {
          if (cs > 1)
            for (int q = 0; q < cs; ++q) s[j] += cluster_map(part, q)[m * RP + c];
          else
            s[j] = part[m * RP + c];
        }
        s[j] *= scale;
        top = fmaxf(top, fabsf(s[j]));
      }
      if constexpr (std::is_same<T, __half>::value) {
        // f16: the row is brought near 1 by a power of two, since t may lie beyond f16's range and its low part below it
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float by = __uint_as_float(__float_as_uint(top) & 0x7f800000u);
        if (by == 0.f || by == INFINITY) by = 1.f;
        if (lane == 0) {
          if (FUSED)
            row_by[m] = by;
          else if (m < rows)
            p.t_by[row0 + m] = by;
        }
#pragma unroll
        for (int j = 0; j < VL; ++j) s[j] *= 1.f / by;
      }
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int c = lane + 32 * j;
        if (c < RP) {
          const T h = from_f32<T>(s[j]);
          const float rest = s[j] - to_f32(h);
          const T l = from_f32<T>(fabsf(to_f32(h)) < INFINITY ? rest : 0.f);
          if (FUSED) {
            *reinterpret_cast<T*>(hi + m * S::RPP + c * 2) = h;
            *reinterpret_cast<T*>(lo + m * S::RPP + c * 2) = l;
          }
          if (p.t && (!FUSED || m % cs == rank) && m < rows && c < p.r) {
            T* const to = reinterpret_cast<T*>(p.t) + (int64_t)(row0 + m) * p.r + c;
            to[0] = h;
            to[(int64_t)p.n_rows * p.r] = l;
          }
        }
      }
    }
    __syncwarp();
    if (cs > 1) cluster_arrive();  // the others' parts have been read
    for (int i = nk; i < nk + nn; ++i) {
      cp_wait<S::STAGES - 2>();
      __syncthreads();
      issue(i + S::STAGES - 1);
      unsigned char* const ys = ring + (i % S::STAGES) * S::STAGE;
      const int c0 = (n_first + i - nk) * S::KC;
      constexpr int NT = S::KC / S::WK / 8;
      add_product<T, RP, NT, TRANS>(ys, S::XP, smem_u32(ys) + TM * S::XP, TRANS ? S::XP : S::RPP, hi_at, lo_at, S::RPP, row_by, Y != nullptr,
                                    wm * 16, wk * NT * 8, lane, O + (int64_t)row0 * p.o_sr + c0, p.o_sr, rows, p.N - c0);
    }
    cp_wait<0>();
    __syncthreads();
    if (cs > 1) cluster_wait();
  }
}

constexpr int EXPAND_ROWS = 64, EXPAND_COLS = 128;

template <int RP, bool TRANS>
struct ExpandShape {
  static constexpr int XP = EXPAND_COLS * 2 + 16, RPP = RP * 2 + 16;
  static constexpr int Y = EXPAND_ROWS * XP, V = TRANS ? RP * XP : EXPAND_COLS * RPP;
  static constexpr int BYTES = Y + V + 2 * EXPAND_ROWS * RPP + EXPAND_ROWS * 4;
};

// The second product by itself: a CTA adds t's 64 rows times v's 128 columns to y. All that it reads is asked for at once; what it
// waits for, the other CTAs of its SM work through. It also writes the rows that take nothing (none where out is y).
template <typename T, int RP, bool TRANS>
__global__ void __launch_bounds__(ADAPTER_THREADS, RP <= 32 ? 4 : 2) adapter_expand_kernel(const __grid_constant__ AdapterParams p) {
  using S = ExpandShape<RP, TRANS>;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char *const ys = smem, *const vs = smem + S::Y, *const ts = vs + S::V;
  float* const row_by = reinterpret_cast<float*>(ts + 2 * EXPAND_ROWS * S::RPP);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c_tiles = (p.N + EXPAND_COLS - 1) / EXPAND_COLS;
  const int tile0 = blockIdx.x / c_tiles, c0 = (int)(blockIdx.x % c_tiles) * EXPAND_COLS, b = blockIdx.y;
  const T* const Y = reinterpret_cast<const T*>(p.y);
  T* const O = reinterpret_cast<T*>(p.out);
  constexpr int CH = EXPAND_COLS / 8, RI = ADAPTER_THREADS / CH, RH = RP / 8, TI = ADAPTER_THREADS / RH;
  const int pm = tid / CH, pc = tid % CH * 8, qm = tid / RH, qc = tid % RH * 8;
  pdl_wait();
  pdl_launch_dependents();
  auto bound = [&](int r) { return min(max(r, 0), p.n_rows); };
  auto plain = [&](int r0, int r1, bool nan) {  // rows as they are (y, or 0), or NaN
    if ((p.out == p.y && !nan) || c0 + pc >= p.N) return;
    for (int64_t r = (int64_t)r0 + tile0 * RI + pm; r < r1; r += (int64_t)p.tiles * RI) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (nan) v = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      else if (Y) v = *reinterpret_cast<const uint4*>(Y + r * p.y_sr + c0 + pc);
      *reinterpret_cast<uint4*>(O + r * p.o_sr + c0 + pc) = v;
    }
  };
  if (b == p.B) {  // rows of no sequence
    plain(0, bound(p.start[0]), false);
    plain(bound(p.start[p.B]), p.n_rows, false);
    return;
  }
  const int r0 = bound(p.start[b]), r1 = bound(p.start[b + 1]);
  const int a = p.which[b];
  if (a < 0 || a >= p.n_adapters) {
    plain(r0, r1, a != -1);
    return;
  }
  const T* const V = reinterpret_cast<const T*>(p.v) + (int64_t)a * p.r * p.N;
  const uint32_t y_to = smem_u32(ys) + pm * S::XP + pc * 2, v_at = smem_u32(vs), t_to = smem_u32(ts) + qm * S::RPP + qc * 2;
  const bool column = c0 + pc < p.N;
  for (int row0 = r0 + tile0 * EXPAND_ROWS; row0 < r1; row0 += p.tiles * EXPAND_ROWS) {
    const int rows = min(EXPAND_ROWS, r1 - row0);
    if (Y && column) {  // (places beyond the rows and the columns do not matter)
      const T* const from = Y + (int64_t)(row0 + pm) * p.y_sr + c0 + pc;
#pragma unroll
      for (int q = 0; q < EXPAND_ROWS / RI; ++q)
        if (pm + q * RI < rows) cp16(y_to + q * RI * S::XP, from + q * RI * p.y_sr);
    }
    if (TRANS) {  // by rank, columns contiguous; what lies beyond the rank is 0
      for (int m = pm; m < RP; m += RI) {
        const bool real = m < p.r && column;
        cp16(v_at + m * S::XP + pc * 2, real ? V + (int64_t)m * p.N + c0 + pc : V, real);
      }
    } else {
      for (int m = qm; m < EXPAND_COLS; m += TI) {
        const bool real = qc < p.r && c0 + m < p.N;
        cp16(v_at + m * S::RPP + qc * 2, real ? V + (int64_t)(c0 + m) * p.r + qc : V, real);
      }
    }
    const T* const t = reinterpret_cast<const T*>(p.t);
    for (int m = qm; m < EXPAND_ROWS; m += TI) {
      const bool real = qc < p.r && m < rows;
      const T* const from = real ? t + (int64_t)(row0 + m) * p.r + qc : t;
      cp16(t_to + (m - qm) * S::RPP, from, real);
      cp16(t_to + (EXPAND_ROWS + m - qm) * S::RPP, real ? from + (int64_t)p.n_rows * p.r : t, real);
    }
    if (std::is_same<T, __half>::value && tid < rows) row_by[tid] = p.t_by[row0 + tid];
    cp_commit();
    cp_wait<0>();
    __syncthreads();
    constexpr int NT = EXPAND_COLS / 2 / 8;
    const uint32_t hi = smem_u32(ts);
    add_product<T, RP, NT, TRANS>(ys, S::XP, v_at, TRANS ? S::XP : S::RPP, hi, hi + EXPAND_ROWS * S::RPP, S::RPP, row_by, Y != nullptr,
                                  warp % 4 * 16, warp / 4 * NT * 8, lane, O + (int64_t)row0 * p.o_sr + c0, p.o_sr, rows, p.N - c0);
    __syncthreads();
  }
}

struct AdapterGradParams {
  const void *x, *dy;  // rows (n, K) and (n, N)
  int64_t x_sr, d_sr;
  const void *t, *u;   // (2, n, r): high and low parts of s x A^T and of s dy B
  void *da, *db;       // (n_adapters, r, K) and (n_adapters, N, r); either null
  const int32_t *start, *which;
  int n_rows, B, K, N, r, n_adapters;
};

constexpr int GRAD_MC = 64;     // columns of a CTA
constexpr int GRAD_ROWS = 64;   // rows of a stage
constexpr int GRAD_BATCH = 128; // sequences looked at together

template <int RP>
struct AdapterGradShape {
  static constexpr int PP = GRAD_MC * 2 + 16, RPP = RP * 2 + 16;
  static constexpr int STAGE = GRAD_ROWS * (PP + 2 * RPP);
  static constexpr int STAGES = RP == 128 ? 3 : 4;
  static constexpr int PART = 2 * GRAD_MC * RP * 4;
  static constexpr int BYTES = STAGES * STAGE + PART;
};

// dA and dB: a CTA takes 64 columns of x or of dy and sums their products with u or t over the rows of all sequences that use its
// adapter; a cluster shares those rows out and meets through distributed shared memory, in the ranks' order. An adapter that nobody
// uses gets zeros.
template <typename T, int RP>
__global__ void __launch_bounds__(ADAPTER_THREADS, RP <= 32 ? 3 : 1) adapter_grad_kernel(const __grid_constant__ AdapterGradParams p) {
  using S = AdapterGradShape<RP>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_which[GRAD_BATCH], s_start[GRAD_BATCH + 1];
  float* const part = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int a = blockIdx.y;
  const int k_tiles = p.da ? (p.K + GRAD_MC - 1) / GRAD_MC : 0;
  int c0 = (int)(blockIdx.x / cs);
  const bool of_a = c0 < k_tiles;
  c0 = (of_a ? c0 : c0 - k_tiles) * GRAD_MC;
  const int C = of_a ? p.K : p.N;
  const T* const R = reinterpret_cast<const T*>(of_a ? p.x : p.dy);
  const int64_t sr = of_a ? p.x_sr : p.d_sr;
  const T* const W = reinterpret_cast<const T*>(of_a ? p.u : p.t);
  const uint32_t ring_at = smem_u32(smem);
  const int wm = warp & 3, wk = warp >> 2;  // warps by columns, and by rows of a stage
  pdl_wait();
  pdl_launch_dependents();

  // this CTA's next rows: (first, count), count 0 at the end. All threads walk alike.
  int b = 0, row = 0, row_end = 0, turn = 0;
  auto next = [&](int& first) {
    while (true) {
      while (row >= row_end) {
        if (b >= p.B) return 0;
        const int j = b % GRAD_BATCH;
        if (j == 0) {
          __syncthreads();
          if (tid < GRAD_BATCH && b + tid < p.B) s_which[tid] = p.which[b + tid];
          for (int i = tid; i < GRAD_BATCH + 1 && b + i <= p.B; i += ADAPTER_THREADS)
            s_start[i] = min(max(p.start[b + i], 0), p.n_rows);
          __syncthreads();
        }
        if (s_which[j] == a) {
          row = s_start[j];
          row_end = s_start[j + 1];
        }
        ++b;
      }
      first = row;
      const int n = min(GRAD_ROWS, row_end - row);
      row += GRAD_ROWS;
      if (turn++ % cs == rank) return n;
    }
  };
  int issued = 0, taken = 0;
  bool more = true;
  // a thread's pieces of a stage
  constexpr int CH = GRAD_MC / 8, RI = ADAPTER_THREADS / CH, RH = RP / 8, TI = ADAPTER_THREADS / RH;
  const int pm = tid / CH, pc = tid % CH * 8, qm = tid / RH, qc = tid % RH * 8;
  const uint32_t row_to = ring_at + pm * S::PP + pc * 2, t_to = ring_at + GRAD_ROWS * S::PP + qm * S::RPP + qc * 2;
  const bool column = c0 + pc < C, whole = c0 + GRAD_MC <= C && p.r == RP;
  const int64_t lo_step = (int64_t)p.n_rows * p.r;
  auto issue = [&]() {
    int first = 0;
    const int n = more ? next(first) : 0;
    more = n > 0;
    if (more) {
      const uint32_t stage = (issued % S::STAGES) * S::STAGE;
      const T* const from = R + (int64_t)(first + pm) * sr + c0 + pc;
      const T* const w = W + (int64_t)(first + qm) * p.r + qc;
      if (n == GRAD_ROWS && whole) {
#pragma unroll
        for (int q = 0; q < GRAD_ROWS / RI; ++q) cp16(row_to + stage + q * RI * S::PP, from + q * RI * sr);
#pragma unroll
        for (int q = 0; q < (GRAD_ROWS + TI - 1) / TI; ++q)
          if (GRAD_ROWS % TI == 0 || qm + q * TI < GRAD_ROWS) {
            cp16(t_to + stage + q * TI * S::RPP, w + q * TI * RP);
            cp16(t_to + stage + (GRAD_ROWS + q * TI) * S::RPP, w + q * TI * RP + lo_step);
          }
      } else {
        for (int q = 0; q < GRAD_ROWS / RI; ++q) {
          const bool real = pm + q * RI < n && column;
          cp16(row_to + stage + q * RI * S::PP, real ? from + q * RI * sr : R, real);
        }
        for (int q = 0; q < (GRAD_ROWS + TI - 1) / TI; ++q) {
          const bool real = qm + q * TI < min(n, GRAD_ROWS) && qc < p.r;
          const T* const at = real ? w + (int64_t)q * TI * p.r : W;
          if (qm + q * TI < GRAD_ROWS) {
            cp16(t_to + stage + q * TI * S::RPP, at, real);
            cp16(t_to + stage + (GRAD_ROWS + q * TI) * S::RPP, real ? at + lo_step : W, real);
          }
        }
      }
      ++issued;
    }
    cp_commit();
  };
  float acc[RP / 8][4];
#pragma unroll
  for (int n = 0; n < RP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; ++i) issue();
  while (taken < issued) {
    cp_wait<S::STAGES - 2>();
    __syncthreads();
    issue();
    const uint32_t ps = ring_at + (taken % S::STAGES) * S::STAGE, ts = ps + GRAD_ROWS * S::PP;
    ++taken;
#pragma unroll
    for (int kk = 0; kk < GRAD_ROWS / 32; ++kk) {
      const int k0 = (kk * 2 + wk) * 16;
      // the columns as the product's rows: 16 x 16 of the stage's rows (k) by columns (m), transposed
      uint32_t pa[4];
      ldsm4t(pa, ps + (k0 + (lane >> 4) * 8 + (lane & 7)) * S::PP + (wm * 16 + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
      for (int n = 0; n < RP / 16; ++n) {
        uint32_t h[4], l[4];
        load_b<true>(h, ts, S::RPP, n * 16, k0, lane);
        load_b<true>(l, ts + GRAD_ROWS * S::RPP, S::RPP, n * 16, k0, lane);
        mma16<T>(acc[2 * n], pa, h[0], h[1]);
        mma16<T>(acc[2 * n + 1], pa, h[2], h[3]);
        mma16<T>(acc[2 * n], pa, l[0], l[1]);
        mma16<T>(acc[2 * n + 1], pa, l[2], l[3]);
      }
    }
  }
  {
    const int m = wk * GRAD_MC + wm * 16 + lane / 4, c = (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < RP / 8; ++n) {
      *reinterpret_cast<float2*>(part + m * RP + n * 8 + c) = make_float2(acc[n][0], acc[n][1]);
      *reinterpret_cast<float2*>(part + (m + 8) * RP + n * 8 + c) = make_float2(acc[n][2], acc[n][3]);
    }
  }
  if (cs > 1)
    cluster_sync_all();
  else
    __syncthreads();
  // each CTA finishes a share of the columns: dA as [r][K], dB as [N][r]
  const int m0 = GRAD_MC * rank / cs, m1 = GRAD_MC * (rank + 1) / cs, per = m1 - m0;
  for (int i = tid; i < per * p.r; i += ADAPTER_THREADS) {
    const int m = m0 + (of_a ? i % per : i / p.r), c = of_a ? i / per : i % p.r;
    float s = 0.f;
    for (int q = 0; q < cs; ++q) {
      const float* const from = (cs > 1 ? cluster_map(part, q) : part) + m * RP + c;
      s += from[0] + from[GRAD_MC * RP];
    }
    if (c0 + m < C) {
      if (of_a)
        reinterpret_cast<T*>(p.da)[((int64_t)a * p.r + c) * p.K + c0 + m] = from_f32<T>(s);
      else
        reinterpret_cast<T*>(p.db)[((int64_t)a * p.N + c0 + m) * p.r + c] = from_f32<T>(s);
    }
  }
  __syncwarp();
  if (cs > 1) cluster_sync_all();  // the others have read this CTA's part
}

}  // namespace ta
