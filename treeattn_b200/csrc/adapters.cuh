// Low-rank adapters of many requests beside a shared projection, forward and backward.
//   t = s_a x A_a^T,  out = y + t B_a^T                      on the rows of each sequence, a = which[sequence]
//   u = s_a dy B_a,   dx = u A_a,  dA_a = u^T x,  dB_a = dy^T t   (sums over the rows of all sequences with adapter a)
// A rank of 8 to 128 gives each element of x and y 2 r operations for its 2 bytes: below the 250 an element that the memory allows the
// tensor cores, so the kernels are bound by the rows' bytes (by latency where there are few rows). That is why they use the
// warp-level matrix instruction, whose fragments come from rows of any length: t's sum over the columns of x and its product with B
// are one kernel, x and y are read once and t never leaves the SM (the training form saves it for dB).
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
  int tiles;          // of a sequence that the grid has clusters for
  void* t_out;        // null, or (2, n, r) bf16: t's high and low parts
};

constexpr int ADAPTER_THREADS = 128;
constexpr int ADAPTER_STAGES = 4;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {  // zeros where there is nothing to read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
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

// The B operand's 16 x 16 block (k k0.., n n0..), from n-major rows (k contiguous) or, TR, from k-major ones. pitch in bytes.
template <bool TR>
__device__ __forceinline__ void load_b(uint32_t (&b)[4], uint32_t base, int pitch, int n0, int k0, int lane) {
  if (TR)
    ldsm4t(b, base + (k0 + (lane & 15)) * pitch + (n0 + (lane >> 4) * 8) * 2);
  else
    ldsm4(b, base + (n0 + (lane >> 4) * 8 + (lane & 7)) * pitch + (k0 + ((lane >> 3) & 1) * 8) * 2);
}

template <int TM, int RP, bool TRANS>
struct AdapterShape {
  static constexpr int WM = TM / 16, WK = 4 / WM;    // warps by rows, and by columns of x
  static constexpr int KC = TM == 16 ? 128 : 64;     // columns of x, and of the output, in a stage
  static constexpr int XP = KC * 2 + 16, RPP = RP * 2 + 16;  // pitches of rows by columns and by rank
  static constexpr int F = TRANS ? KC * RPP : RP * XP;       // a stage's part of u, ...
  static constexpr int G = TRANS ? RP * XP : KC * RPP;       // ... and of v
  static constexpr int STAGE = TM * XP + (F > G ? F : G);
  static constexpr int PART = 4 / WM * TM * RP * 4;
  static constexpr int BYTES = ADAPTER_STAGES * STAGE + PART + 2 * TM * RPP + TM * 4;
};

// A cluster of CTAs takes a tile of a sequence's rows. Each contracts a share of x's columns; the partial t meet through distributed
// shared memory (summed in the ranks' order by each CTA for itself) and each CTA adds its share of the output's columns. The stages of
// both halves go through one ring of asynchronous copies, so that the second half's first stages arrive while t is summed.
// Tiles of 16 rows serve decoding, of 64 rows prompts and training.
template <typename T, int TM, int RP, bool TRANS>
__global__ void __launch_bounds__(ADAPTER_THREADS) adapter_kernel(const __grid_constant__ AdapterParams p) {
  using S = AdapterShape<TM, RP, TRANS>;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const ring = smem;
  float* const part = reinterpret_cast<float*>(smem + ADAPTER_STAGES * S::STAGE);
  unsigned char* const hi = smem + ADAPTER_STAGES * S::STAGE + S::PART;
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
    if (p.out == p.y && !nan) return;
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
  const int n_first = nc * rank / cs, nn = nc * (rank + 1) / cs - n_first;
  const uint32_t ring_at = smem_u32(ring), hi_at = smem_u32(hi), lo_at = smem_u32(lo);
  constexpr int CH = S::KC / 8, RH = RP / 8;  // 16-byte pieces of a row by columns, by rank

  for (int row0 = r0 + tile0 * TM; row0 < r1; row0 += p.tiles * TM) {
    const int rows = min(TM, r1 - row0);
    auto issue = [&](int i) {
      if (i < nk + nn) {
        const bool first = i < nk;
        const uint32_t at = ring_at + (i % ADAPTER_STAGES) * S::STAGE;
        const int c0 = (first ? k_first + i : n_first + i - nk) * S::KC, C = first ? p.K : p.N;
        const T* const R = first ? X : Y;
        const int64_t sr = first ? p.x_sr : p.y_sr;
        if (R)
          for (int j = tid; j < TM * CH; j += ADAPTER_THREADS) {
            const int m = j / CH, c = j % CH * 8;
            const bool real = m < rows && c0 + c < C;
            cp16(at + m * S::XP + c * 2, real ? R + (int64_t)(row0 + m) * sr + c0 + c : R, real);
          }
        // the factor's part: by rank, columns contiguous (u forward, v TRANS), or by column, rank contiguous
        const T* const W = first ? U : V;
        const uint32_t to = at + TM * S::XP;
        if (first != TRANS) {
          for (int j = tid; j < RP * CH; j += ADAPTER_THREADS) {
            const int m = j / CH, c = j % CH * 8;
            const bool real = m < p.r && c0 + c < C;
            cp16(to + m * S::XP + c * 2, real ? W + (int64_t)m * C + c0 + c : W, real);
          }
        } else {
          for (int j = tid; j < S::KC * RH; j += ADAPTER_THREADS) {
            const int m = j / RH, c = j % RH * 8;
            const bool real = c < p.r && c0 + m < C;
            cp16(to + m * S::RPP + c * 2, real ? W + (int64_t)(c0 + m) * p.r + c : W, real);
          }
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < ADAPTER_STAGES - 1; ++i) issue(i);

    float acc[RP / 8][4];
#pragma unroll
    for (int n = 0; n < RP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    for (int i = 0; i < nk; ++i) {
      cp_wait<ADAPTER_STAGES - 2>();
      __syncthreads();
      issue(i + ADAPTER_STAGES - 1);
      const uint32_t xs = ring_at + (i % ADAPTER_STAGES) * S::STAGE, us = xs + TM * S::XP;
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
    for (int m = warp; m < TM; m += ADAPTER_THREADS / 32) {
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
        if (lane == 0) row_by[m] = by;
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
          *reinterpret_cast<T*>(hi + m * S::RPP + c * 2) = h;
          *reinterpret_cast<T*>(lo + m * S::RPP + c * 2) = l;
          if (p.t_out && m % cs == rank && m < rows && c < p.r) {
            T* const to = reinterpret_cast<T*>(p.t_out) + (int64_t)(row0 + m) * p.r + c;
            to[0] = h;
            to[(int64_t)p.n_rows * p.r] = l;
          }
        }
      }
    }
    __syncwarp();
    if (cs > 1) cluster_arrive();  // the others' parts have been read
    constexpr int NT = S::KC / S::WK / 8;  // a warp's tiles of 8 columns
    for (int i = nk; i < nk + nn; ++i) {
      cp_wait<ADAPTER_STAGES - 2>();
      __syncthreads();
      issue(i + ADAPTER_STAGES - 1);
      unsigned char* const ys = ring + (i % ADAPTER_STAGES) * S::STAGE;
      const uint32_t vs = smem_u32(ys) + TM * S::XP;
      float o[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < RP / 16; ++kk) {
        uint32_t th[4], tl[4];
        const uint32_t at = (wm * 16 + (lane & 15)) * S::RPP + (kk * 16 + (lane >> 4) * 8) * 2;
        ldsm4(th, hi_at + at);
        ldsm4(tl, lo_at + at);
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          uint32_t vb[4];
          load_b<TRANS>(vb, vs, TRANS ? S::XP : S::RPP, wk * NT * 8 + n * 16, kk * 16, lane);
          mma16<T>(o[2 * n], th, vb[0], vb[1]);
          mma16<T>(o[2 * n + 1], th, vb[2], vb[3]);
          mma16<T>(o[2 * n], tl, vb[0], vb[1]);
          mma16<T>(o[2 * n + 1], tl, vb[2], vb[3]);
        }
      }
      // added to y where it lies, rounded once; whole 16-byte pieces then leave
      const int c0 = (n_first + i - nk) * S::KC;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int m = wm * 16 + lane / 4 + 8 * h;
        const float by = std::is_same<T, __half>::value ? row_by[m] : 1.f;
        unsigned char* const at = ys + m * S::XP + (wk * NT * 8 + (lane & 3) * 2) * 2;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          T* const e = reinterpret_cast<T*>(at + n * 16);
          const float y0 = Y ? to_f32(e[0]) : 0.f, y1 = Y ? to_f32(e[1]) : 0.f;
          e[0] = from_f32<T>(fmaf(o[n][2 * h], by, y0));
          e[1] = from_f32<T>(fmaf(o[n][2 * h + 1], by, y1));
        }
      }
      __syncwarp();
      for (int j = lane; j < 16 * NT; j += 32) {
        const int m = wm * 16 + j / NT, c = wk * NT * 8 + j % NT * 8;
        if (m < rows && c0 + c < p.N)
          *reinterpret_cast<uint4*>(O + (int64_t)(row0 + m) * p.o_sr + c0 + c) = *reinterpret_cast<const uint4*>(ys + m * S::XP + c * 2);
      }
    }
    cp_wait<0>();
    __syncthreads();
    if (cs > 1) cluster_wait();
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
  static constexpr int PART = GRAD_MC * RP * 4;
  static constexpr int BYTES = STAGES * STAGE + PART;
};

// dA and dB: a CTA takes 64 columns of x or of dy and sums their products with u or t over the rows of all sequences that use its
// adapter; a cluster shares those rows out and meets through distributed shared memory, in the ranks' order. An adapter that nobody
// uses gets zeros.
template <typename T, int RP>
__global__ void __launch_bounds__(ADAPTER_THREADS) adapter_grad_kernel(const __grid_constant__ AdapterGradParams p) {
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
          if (b + tid < p.B) s_which[tid] = p.which[b + tid];
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
  auto issue = [&]() {
    int first = 0;
    const int n = more ? next(first) : 0;
    more = n > 0;
    if (more) {
      const uint32_t at = ring_at + (issued % S::STAGES) * S::STAGE;
      for (int j = tid; j < GRAD_ROWS * (GRAD_MC / 8); j += ADAPTER_THREADS) {
        const int m = j / (GRAD_MC / 8), c = j % (GRAD_MC / 8) * 8;
        const bool real = m < n && c0 + c < C;
        cp16(at + m * S::PP + c * 2, real ? R + (int64_t)(first + m) * sr + c0 + c : R, real);
      }
      for (int j = tid; j < 2 * GRAD_ROWS * (RP / 8); j += ADAPTER_THREADS) {
        const int m = j / (RP / 8), c = j % (RP / 8) * 8, half = m / GRAD_ROWS, mm = m % GRAD_ROWS;
        const bool real = mm < n && c < p.r;
        cp16(at + GRAD_ROWS * S::PP + m * S::RPP + c * 2,
             real ? W + ((int64_t)half * p.n_rows + first + mm) * p.r + c : W, real);
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
    for (int k0 = 0; k0 < GRAD_ROWS; k0 += 16) {
      // the columns as the product's rows: 16 x 16 of the stage's rows (k) by columns (m), transposed
      uint32_t pa[4];
      ldsm4t(pa, ps + (k0 + (lane >> 4) * 8 + (lane & 7)) * S::PP + (warp * 16 + ((lane >> 3) & 1) * 8) * 2);
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
    const int m = warp * 16 + lane / 4, c = (lane & 3) * 2;
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
    for (int q = 0; q < cs; ++q) s += (cs > 1 ? cluster_map(part, q) : part)[m * RP + c];
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
