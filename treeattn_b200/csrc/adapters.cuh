// Low-rank adapters of many requests beside a shared projection, forward and backward.
//   t = s_a x A_a^T,  out = y + t B_a^T                      on the rows of each sequence, a = which[sequence]
//   u = s_a dy B_a,   dx = u A_a,  dA_a = u^T x,  dB_a = dy^T t   (sums over the rows of all sequences with adapter a)
// A rank of 8 to 128 gives each element of x and y 2 r operations for its 2 bytes: below the 250 an element that the memory allows the
// tensor cores, so the kernels are bound by the rows' bytes (by latency where there are few rows). That is why they use the
// warp-level matrix instruction, whose fragments come from rows of any length.
// Few rows of a sequence (decoding) take one kernel for both products; many take two, t going by way of memory (64 bytes a row at rank
// 16): its columns and the output's are then shared out over the GPU apart.
// t is held in fp32 and enters its product as two 16-bit numbers, high and low: 16 bits of it (22 in f16; see split), so that the output's one
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

// The B operand's 16 x 16 block (n n0.., k k0..) from rows by n with k contiguous; pitch in bytes.
__device__ __forceinline__ void load_b(uint32_t (&b)[4], uint32_t base, int pitch, int n0, int k0, int lane) {
  ldsm4(b, base + (n0 + (lane >> 4) * 8 + (lane & 7)) * pitch + (k0 + ((lane >> 3) & 1) * 8) * 2);
}

// s as two 16-bit numbers of one sign, h the next below s in magnitude (toward 0), l the rest, neither of them 0 where s is not: a factor
// that is infinite then gives the infinity of s times it, and not the NaN of infinities of both signs or of 0 times one. l is rounded once, by
// 2^-16 of s at most (bf16; f16 2^-22). An infinite s goes on as inf + 1. (bf16 numbers below 2^-132 keep h or l alone.)
__device__ __forceinline__ void split(float s, __nv_bfloat16& h, __nv_bfloat16& l) {
  const uint32_t u = __float_as_uint(s), mag = u & 0x7fffffffu;
  const bool some = mag - 1u < 0x7f7fffffu;  // finite and not 0
  const float f = some ? __uint_as_float((u - 1u) & 0xffff0000u) : s;
  const float rest = some ? s - f : (mag == 0x7f800000u ? copysignf(1.f, s) : 0.f);
  h = from_f32<__nv_bfloat16>(f);
  l = from_f32<__nv_bfloat16>(rest);
}
// f16, |s| below 2 but in rows that hold an infinity or are below 2^-126 whole: there l ends at 65504, and s up to 2^-24 is l alone, as
// elsewhere. Beside an h that is not 0 l is 2^-24 at least.
__device__ __forceinline__ void split(float s, __half& h, __half& l) {
  h = __float2half_rz(s);
  l = __float2half_rn(0.f);
  if (fabsf(s) == INFINITY) {
    l = __float2half_rn(copysignf(1.f, s));
  } else if (fabsf(s) > 0.f) {
    const uint16_t b = __half_as_ushort(h);
    if ((b & 0x7fffu) && __half2float(h) == s) h = __ushort_as_half((uint16_t)(b - 1u));
    const float t = __half2float(h), rest = fminf(fabsf(s - t), 65504.f);
    l = __float2half_rn(copysignf(t == 0.f ? rest : fmaxf(rest, 5.9604644775390625e-08f), s));
  }
}

// A warp's row m of t: summed over the cluster's parts (rows of RP), scaled, split into high and low parts. They go to p.t's row `row`
// (unless there is none), and to shared memory where that is given.
template <typename T, int RP>
__device__ __forceinline__ void split_row(const AdapterParams& p, const float* part, int cs, int m, int row, float scale, int lane,
                                          unsigned char* hi = nullptr, unsigned char* lo = nullptr, float* by_out = nullptr) {
  constexpr int VL = (RP + 31) / 32;
  float s[VL], top = 0.f, by = 1.f;
#pragma unroll
  for (int v = 0; v < VL; ++v) {
    const int c = lane + 32 * v;
    s[v] = 0.f;
    if (c < p.r) {  // (ranks that fill it up stay 0: an infinity in x times their zeros would be NaN)
      if (cs > 1)
        for (int q = 0; q < cs; ++q) s[v] += cluster_map(part, q)[m * RP + c];
      else
        s[v] = part[m * RP + c];
    }
    s[v] *= scale;
    top = fmaxf(top, fabsf(s[v]));
  }
  if constexpr (std::is_same<T, __half>::value) {
    // f16: the row is brought near 1 by a power of two, since t may lie beyond f16's range and its low part below it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    by = __uint_as_float(__float_as_uint(top) & 0x7f800000u);
    if (by == 0.f || by == INFINITY) by = 1.f;
#pragma unroll
    for (int v = 0; v < VL; ++v) s[v] *= 1.f / by;
    if (p.t && row >= 0 && lane == 0) p.t_by[row] = by;
  }
  if (by_out) *by_out = by;
#pragma unroll
  for (int v = 0; v < VL; ++v) {
    const int c = lane + 32 * v;
    if (c >= RP) break;
    T h, l;
    split(s[v], h, l);
    if (hi) {
      reinterpret_cast<T*>(hi)[c] = h;
      reinterpret_cast<T*>(lo)[c] = l;
    }
    if (p.t && row >= 0 && c < p.r) {
      T* const to = reinterpret_cast<T*>(p.t) + (int64_t)row * p.r + c;
      to[0] = h;
      to[(int64_t)p.n_rows * p.r] = l;
    }
  }
}

// ------------------------------------------------------------------------------------------------ few rows
template <int RP>
struct AdapterShape {
  static constexpr int KC = 128;                             // columns of x, and of the output, in a stage
  static constexpr int STAGES = 3;
  static constexpr int XP = KC * 2 + 16, RPP = RP * 2 + 16;  // pitches of rows by columns and by rank
  static constexpr int U = RP * XP, V = KC * RPP;            // a stage's part of the factors
  static constexpr int STAGE = 16 * XP + (U > V ? U : V);
  static constexpr int PART = 8 * 16 * RP * 4;
  static constexpr int BYTES = STAGES * STAGE + PART + 2 * 16 * RPP + 16 * 4;
};

// Both products of 16 rows of a sequence by one cluster of CTAs. Each contracts a share of x's columns (its warps by sixteens); the partial
// t meet through distributed shared memory, summed in the ranks' order by each CTA for itself, and each adds its share of the
// output's columns. The stages of both halves go through one ring of asynchronous copies, so that the second half's first stages arrive
// while t is summed. Bound by latency: a chain of copy, product, cluster barrier, product; one row of 2048 -> 2048 at rank 8 takes 5 us, 64
// sequences' rows of 768 -> 2304 at rank 16 take 8 (weights in the L2).
template <typename T, int RP>
__global__ void __launch_bounds__(ADAPTER_THREADS, RP <= 32 ? 4 : RP == 64 ? 2 : 1)
    adapter_kernel(const __grid_constant__ AdapterParams p) {
  using S = AdapterShape<RP>;
  extern __shared__ __align__(16) unsigned char smem[];
  float* const part = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE);
  unsigned char* const hi = smem + S::STAGES * S::STAGE + S::PART;
  unsigned char* const lo = hi + 16 * S::RPP;
  float* const row_by = reinterpret_cast<float*>(lo + 16 * S::RPP);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int tile0 = blockIdx.x / cs, b = blockIdx.y;
  const T* const X = reinterpret_cast<const T*>(p.x);
  const T* const Y = reinterpret_cast<const T*>(p.y);
  T* const O = reinterpret_cast<T*>(p.out);
  pdl_wait();
  pdl_launch_dependents();

  auto plain = [&](int r0, int r1, bool nan) {  // rows as they are, or NaN
    if (p.out == p.y && !nan) return;
    const int pieces = p.N / 8;
    for (int64_t i = (int64_t)blockIdx.x * ADAPTER_THREADS + tid; i < (int64_t)(r1 - r0) * pieces;
         i += (int64_t)gridDim.x * ADAPTER_THREADS) {
      const int64_t row = r0 + i / pieces;
      const int c = (int)(i % pieces) * 8;
      uint4 v = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      if (!nan) v = *reinterpret_cast<const uint4*>(Y + row * p.y_sr + c);
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
  const int kc = (p.K + S::KC - 1) / S::KC, nc = (p.N + S::KC - 1) / S::KC;
  const int k_first = kc * rank / cs, nk = kc * (rank + 1) / cs - k_first;
  const int n_first = nc * rank / cs, nn = nc * (rank + 1) / cs - n_first;
  const uint32_t ring_at = smem_u32(smem), hi_at = smem_u32(hi);
  // a thread's pieces of a stage: a row's columns (16 of its 16 rows' 256 bytes), a column's ranks
  constexpr int CH = S::KC / 8, RH = RP / 8, CI = ADAPTER_THREADS / RH;
  static_assert(ADAPTER_THREADS / CH == 16, "a row of threads for each row");
  const int pm = tid / CH, pc = tid % CH * 8, qm = tid / RH, qc = tid % RH * 8;
  const uint32_t row_to = ring_at + pm * S::XP + pc * 2, col_to = ring_at + 16 * S::XP + qm * S::RPP + qc * 2;
  const bool whole_rank = p.r == RP;

  for (int row0 = r0 + tile0 * 16; row0 < r1; row0 += p.tiles * 16) {
    const int rows = min(16, r1 - row0);
    const T* const x_at = X + (int64_t)(row0 + pm) * p.x_sr + pc;
    const T* const y_at = Y + (int64_t)(row0 + pm) * p.y_sr + pc;
    auto issue = [&](int i) {
      if (i < nk + nn) {
        const bool first = i < nk;
        const uint32_t stage = (i % S::STAGES) * S::STAGE;
        const int c0 = (first ? k_first + i : n_first + i - nk) * S::KC, C = first ? p.K : p.N;
        const bool cut = c0 + S::KC > C;  // the columns end in this stage: x's and u's are filled up with zeros, y's do not matter
        if (pm < rows) {                  // (the places of rows that are not there keep what they hold)
          const bool real = c0 + pc < C;
          cp16(row_to + stage, real ? (first ? x_at : y_at) + c0 : X, real);
        }
        if (first) {
          const T* const w = U + (int64_t)pm * C + c0 + pc;
#pragma unroll
          for (int q = 0; q < RP / 16; ++q) {
            const bool real = pm + 16 * q < p.r && c0 + pc < C;
            cp16(row_to + 16 * S::XP + stage + q * 16 * S::XP, real ? w + (int64_t)q * 16 * C : U, real);
          }
        } else {
          const T* const w = V + (int64_t)(c0 + qm) * p.r + qc;
          if (!cut && whole_rank) {
#pragma unroll
            for (int q = 0; q < (S::KC + CI - 1) / CI; ++q)
              if (S::KC % CI == 0 || qm + q * CI < S::KC) cp16(col_to + stage + q * CI * S::RPP, w + q * CI * RP);
          } else {
            for (int q = 0; q < (S::KC + CI - 1) / CI; ++q) {
              const bool real = qc < p.r && c0 + qm + q * CI < C;
              if (qm + q * CI < S::KC) cp16(col_to + stage + q * CI * S::RPP, real ? w + (int64_t)q * CI * p.r : V, real);
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
      const uint32_t xs = ring_at + (i % S::STAGES) * S::STAGE, us = xs + 16 * S::XP;
      uint32_t xa[4];
      ldsm4(xa, xs + (lane & 15) * S::XP + (warp * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
      for (int n = 0; n < RP / 16; ++n) {
        uint32_t ub[4];
        load_b(ub, us, S::XP, n * 16, warp * 16, lane);
        mma16<T>(acc[2 * n], xa, ub[0], ub[1]);
        mma16<T>(acc[2 * n + 1], xa, ub[2], ub[3]);
      }
    }
    // the warps' parts, the CTA's, the cluster's
    {
      float* const to = part + (warp * 16 + lane / 4) * RP + (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < RP / 8; ++n) {
        *reinterpret_cast<float2*>(to + n * 8) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(to + 8 * RP + n * 8) = make_float2(acc[n][2], acc[n][3]);
      }
    }
    __syncthreads();
    for (int i = tid; i < 16 * RP; i += ADAPTER_THREADS) {
      float s = part[i];
#pragma unroll
      for (int w = 1; w < 8; ++w) s += part[w * 16 * RP + i];
      part[i] = s;
    }
    if (cs > 1)
      cluster_sync_all();
    else
      __syncthreads();
    for (int m = warp; m < 16; m += 8) {
      float by;
      split_row<T, RP>(p, part, cs, m, m < rows && m % cs == rank ? row0 + m : -1, scale, lane, hi + m * S::RPP, lo + m * S::RPP, &by);
      if (lane == 0) row_by[m] = by;
    }
    __syncwarp();
    if (cs > 1) cluster_arrive();  // the others' parts have been read
    const uint32_t t_at = hi_at + (lane & 15) * S::RPP + (lane >> 4) * 16;
    for (int i = nk; i < nk + nn; ++i) {
      cp_wait<S::STAGES - 2>();
      __syncthreads();
      issue(i + S::STAGES - 1);
      unsigned char* const ys = smem + (i % S::STAGES) * S::STAGE;
      const uint32_t y_at16 = smem_u32(ys) + (lane & 15) * S::XP + (warp * 16 + (lane >> 4) * 8) * 2, vs = smem_u32(ys) + 16 * S::XP;
      // a warp's 16 columns
      float o[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kk = 0; kk < RP / 16; ++kk) {
        uint32_t th[4], tl[4], vb[4];
        ldsm4(th, t_at + kk * 32);
        ldsm4(tl, t_at + 16 * S::RPP + kk * 32);
        load_b(vb, vs, S::RPP, warp * 16, kk * 16, lane);
        mma16<T>(o[0], th, vb[0], vb[1]);
        mma16<T>(o[1], th, vb[2], vb[3]);
        mma16<T>(o[0], tl, vb[0], vb[1]);
        mma16<T>(o[1], tl, vb[2], vb[3]);
      }
      // added to y where it lies, rounded once; whole 16-byte pieces then leave
      uint32_t y4[4];
      ldsm4(y4, y_at16);
      const float by[2] = {row_by[lane / 4], row_by[lane / 4 + 8]};
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float2 f = widen2<T>(y4[h]);
        y4[h] = narrow2<T>(fmaf(o[h / 2][h % 2 * 2], by[h % 2], f.x), fmaf(o[h / 2][h % 2 * 2 + 1], by[h % 2], f.y));
      }
      stsm4(y_at16, y4);
      __syncwarp();
      const int m = lane / 2, c = warp * 16 + lane % 2 * 8, c0 = (n_first + i - nk) * S::KC;
      if (m < rows && c0 + c < p.N)
        *reinterpret_cast<uint4*>(O + (int64_t)(row0 + m) * p.o_sr + c0 + c) = *reinterpret_cast<const uint4*>(ys + m * S::XP + c * 2);
    }
    cp_wait<0>();
    __syncthreads();
    if (cs > 1) cluster_wait();
  }
}

// ------------------------------------------------------------------------------------------------ many rows
// t's kernel takes its operands from memory straight into the fragments of the matrix instruction: the order of a sum's
// terms and of an output's columns is free, and it is chosen so that a thread's share of a fragment is 16 consecutive bytes
// of a row. Nothing passes through shared memory but the warps' sums at the end, and no warp waits for another before that.
//   k of a 32-wide block: step s (0, 1), the fragment's pair (lane % 4 = j, half h) <-> elements 8 j + 4 s + 2 h, + 1
//   columns of a 32-wide block: tile q (0 to 3), the fragment's pair j <-> columns 8 j + 2 q, + 1
// Where a factor's rows run the other way an 8 x 8 block is turned in registers.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2& v, int i) { return i == 0 ? v.x : v.y; }
__device__ __forceinline__ uint4 load16(const void* p, bool real) {
  return real ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ uint2 load8(const void* p, bool real) {
  return real ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0u, 0u);
}

template <int RP>
struct ShrinkShape {
  static constexpr int G = RP == 16 ? 1 : RP / 32, KS = 8 / G;      // warps by ranks (at most 32 each), and by columns
  static constexpr int MT = RP <= 32 ? 2 : 4, ROWS = 16 * MT;       // rows of a CTA: more where a factor's row weighs more
  static constexpr int BYTES = KS * ROWS * RP * 4;
};

// t = s x U^T by itself: a CTA takes 32 or 64 rows, its warps (and the CTAs of a cluster) 32 ranks each and every so many blocks of 32
// columns; their sums meet in one order. Bound by the latency of a warp's loads: 16384 rows at rank 16, 768 columns in 12 us (2.1 TB/s), 2304
// turned in 24 us (3.2 TB/s). From shared memory, filled ahead, the first took 14 us and the second 36; at rank 128 the first takes 31 us,
// with a factor's ranks all in one warp it took 110.
template <typename T, int RP, bool TRANS>
__global__ void __launch_bounds__(ADAPTER_THREADS, RP == 16 ? 4 : RP == 32 ? 3 : 2) adapter_shrink_kernel(const __grid_constant__ AdapterParams p) {
  using S = ShrinkShape<RP>;
  constexpr int MT = S::MT, NT = RP / 8 / S::G;
  extern __shared__ __align__(16) float part[];  // (KS, ROWS, RP)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = lane >> 2, j = lane & 3;
  const int rank0 = warp % S::G * 32, ks = warp / S::G;  // the warp's first rank
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int tile0 = blockIdx.x / cs, b = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  auto bound = [&](int r) { return min(max(r, 0), p.n_rows); };
  const int r0 = bound(p.start[b]), r1 = bound(p.start[b + 1]);
  const int a = p.which[b];
  if (a < 0 || a >= p.n_adapters) {
    if (a != -1 && blockIdx.x == 0 && tid == 0) record_error(DEV_INDEX_RANGE, K_ADAPTER, b, a);
    return;
  }
  const T* const U = reinterpret_cast<const T*>(p.u) + (int64_t)a * p.r * p.K;
  const float scale = p.scale ? p.scale[a] : 1.f;
  const int blocks = (p.K + 31) / 32;
  for (int row0 = r0 + tile0 * S::ROWS; row0 < r1; row0 += p.tiles * S::ROWS) {
    const int rows = min(S::ROWS, r1 - row0);
    const T* const x = reinterpret_cast<const T*>(p.x) + (int64_t)(row0 + i) * p.x_sr + 8 * j;
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
#pragma unroll 1
    for (int kb = rank * S::KS + ks; kb < blocks; kb += S::KS * cs) {
      const int k0 = kb * 32;
      const bool in = k0 + 8 * j < p.K;
      uint4 xv[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          xv[m][h] = load16(x + (int64_t)(16 * m + 8 * h) * p.x_sr + k0, in && 16 * m + 8 * h + i < rows);
      uint32_t ub[2][2][NT];  // step, half, tile
      if (!TRANS) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int c = rank0 + 8 * n + i;
          const uint4 u = load16(U + (int64_t)c * p.K + k0 + 8 * j, in && c < p.r);
          ub[0][0][n] = u.x; ub[0][1][n] = u.y; ub[1][0][n] = u.z; ub[1][1][n] = u.w;
        }
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = k0 + 8 * (i >> 1) + 4 * s + 2 * h + (i & 1);
            const T* const row = U + (int64_t)k * p.r + rank0;
            if (RP == 16) {
              const uint2 u = load8(row + 4 * j, k < p.K && 4 * j < p.r);
              ub[s][h][0] = turned(u.x);
              ub[s][h][1] = turned(u.y);
            } else {
              const uint4 u = load16(row + 8 * j, k < p.K && rank0 + 8 * j < p.r);
#pragma unroll
              for (int q = 0; q < NT; ++q) ub[s][h][q] = turned(word(u, q));
            }
          }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint32_t xa[4] = {word(xv[m][0], 2 * s), word(xv[m][1], 2 * s), word(xv[m][0], 2 * s + 1), word(xv[m][1], 2 * s + 1)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16<T>(acc[m][n], xa, ub[s][0][n], ub[s][1][n]);
        }
    }
    // the warps' sums, the CTA's, the cluster's
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int c = rank0 + (!TRANS ? 8 * n + 2 * j : RP == 16 ? 4 * j + 2 * n : 8 * j + 2 * n);
        float* const to = part + (ks * S::ROWS + 16 * m + i) * RP + c;
        *reinterpret_cast<float2*>(to) = make_float2(acc[m][n][0], acc[m][n][1]);
        *reinterpret_cast<float2*>(to + 8 * RP) = make_float2(acc[m][n][2], acc[m][n][3]);
      }
    __syncthreads();
    for (int e = tid; e < S::ROWS * RP; e += ADAPTER_THREADS) {
      float s = part[e];
#pragma unroll
      for (int w = 1; w < S::KS; ++w) s += part[w * S::ROWS * RP + e];
      part[e] = s;
    }
    if (cs > 1)
      cluster_sync_all();
    else
      __syncthreads();
    for (int m = warp * cs + rank; m < rows; m += 8 * cs)
      split_row<T, RP>(p, part, cs, m, row0 + m, scale, lane);
    __syncwarp();
    if (cs > 1)
      cluster_sync_all();  // the others' parts have been read
    else
      __syncthreads();
  }
}

// The output's 16 x 8 NT block of a warp, from y's tile at `tile` (pitch XP): t's rows times v, added, rounded once and written back there;
// whole 16-byte pieces then leave for rows below `rows` and columns below `cols` of `out` (the CTA's corner).
template <typename T, int RP, int NT, bool TRANS>
__device__ __forceinline__ void add_product(unsigned char* tile, int xp, uint32_t vs, int vp, uint32_t hi, uint32_t lo, int tp, const float* row_by,
                                            bool with_y, int m0, int n0, int lane, T* out, int64_t o_sr, int rows, int cols) {
  constexpr bool FROM_Y = !std::is_same<T, __half>::value;  // the sum begins with y (f16's rows have a factor of their own)
  uint32_t y_at = smem_u32(tile) + (m0 + (lane & 15)) * xp + (n0 + (lane >> 4) * 8) * 2;
  const uint32_t t_at = (m0 + (lane & 15)) * tp + (lane >> 4) * 16;
  constexpr int PN = RP <= 32 ? NT / 2 : NT;  // (small ranks in two parts: fewer registers, more warps' loads in flight)
#pragma unroll 1
  for (int part = 0; part < NT; part += PN, y_at += PN * 16, n0 += PN * 8) {
    float o[PN][4];
    auto begin = [&](auto set) {
#pragma unroll
      for (int n = 0; n < PN; n += 2) {
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
      for (int n = 0; n < PN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    }
#pragma unroll
    for (int kk = 0; kk < RP / 16; ++kk) {
      uint32_t th[4], tl[4];
      ldsm4(th, hi + t_at + kk * 32);
      ldsm4(tl, lo + t_at + kk * 32);
#pragma unroll
      for (int n = 0; n < PN / 2; ++n) {
        uint32_t vb[4];
        if (TRANS)
          ldsm4t(vb, vs + (kk * 16 + (lane & 15)) * vp + (n0 + n * 16 + (lane >> 4) * 8) * 2);
        else
          load_b(vb, vs, vp, n0 + n * 16, kk * 16, lane);
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
    for (int n = 0; n < PN; n += 2) {
      const uint32_t r4[4] = {narrow2<T>(o[n][0], o[n][1]), narrow2<T>(o[n][2], o[n][3]), narrow2<T>(o[n + 1][0], o[n + 1][1]),
                              narrow2<T>(o[n + 1][2], o[n + 1][3])};
      stsm4(y_at + n * 16, r4);
    }
  }
  n0 -= NT * 8;
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

constexpr int EXPAND_ROWS = 64, EXPAND_COLS = 128;

template <int RP, bool TRANS>
struct ExpandShape {
  static constexpr int XP = EXPAND_COLS * 2 + 16, RPP = RP * 2 + 16;
  static constexpr int Y = EXPAND_ROWS * XP, V = TRANS ? RP * XP : EXPAND_COLS * RPP;
  static constexpr int BYTES = Y + V + 2 * EXPAND_ROWS * RPP + EXPAND_ROWS * 4;
};

// The second product by itself: a CTA adds t's 64 rows times v's 128 columns to y. All that it reads is asked for at once; what it
// waits for, the other CTAs of its SM work through. It also writes the rows that take nothing (none where out is y). 16384 rows of 2304
// columns, rank 16: 32 us (150 MB read and written, 4.7 TB/s; 34 with four CTAs on an SM instead of six); rank 128: 75 us, the matrix
// instructions (two a product) at half of what they can do. With fragments from memory instead of shared memory: 36 us, and 180 at rank
// 128, where v is read 4 times as often.
template <typename T, int RP, bool TRANS>
__global__ void __launch_bounds__(ADAPTER_THREADS, RP == 16 ? 6 : RP == 32 ? 5 : RP == 64 ? 3 : 2)
    adapter_expand_kernel(const __grid_constant__ AdapterParams p) {
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
  const bool column = c0 + pc < p.N, whole = c0 + EXPAND_COLS <= p.N && p.r == RP;
  const int64_t y_step = RI * p.y_sr, lo_step = (int64_t)p.n_rows * p.r;
  for (int row0 = r0 + tile0 * EXPAND_ROWS; row0 < r1; row0 += p.tiles * EXPAND_ROWS) {
    const int rows = min(EXPAND_ROWS, r1 - row0);
    const T* const t = reinterpret_cast<const T*>(p.t) + (int64_t)(row0 + qm) * p.r + qc;
    if (whole && rows == EXPAND_ROWS) {
      if (Y) {
        const T* from = Y + (int64_t)(row0 + pm) * p.y_sr + c0 + pc;
#pragma unroll
        for (int q = 0; q < EXPAND_ROWS / RI; ++q, from += y_step) cp16(y_to + q * RI * S::XP, from);
      }
#pragma unroll
      for (int q = 0; q < (TRANS ? RP / RI : EXPAND_COLS / TI); ++q) {
        if (TRANS)
          cp16(v_at + (pm + q * RI) * S::XP + pc * 2, V + (int64_t)(pm + q * RI) * p.N + c0 + pc);
        else
          cp16(v_at + (qm + q * TI) * S::RPP + qc * 2, V + (int64_t)(c0 + qm) * RP + qc + q * TI * RP);
      }
#pragma unroll
      for (int q = 0; q < (EXPAND_ROWS + TI - 1) / TI; ++q)
        if (EXPAND_ROWS % TI == 0 || qm < EXPAND_ROWS) {
          cp16(t_to + q * TI * S::RPP, t + q * TI * RP);
          cp16(t_to + (EXPAND_ROWS + q * TI) * S::RPP, t + q * TI * RP + lo_step);
        }
    } else {
      if (Y && column) {  // (places beyond the rows and the columns do not matter)
        const T* const from = Y + (int64_t)(row0 + pm) * p.y_sr + c0 + pc;
        for (int q = 0; q < EXPAND_ROWS / RI; ++q)
          if (pm + q * RI < rows) cp16(y_to + q * RI * S::XP, from + q * y_step);
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
      for (int m = qm; m < EXPAND_ROWS; m += TI) {
        const bool real = qc < p.r && m < rows;
        const T* const from = real ? t + (int64_t)(m - qm) * p.r : V;
        cp16(t_to + (m - qm) * S::RPP, from, real);
        cp16(t_to + (EXPAND_ROWS + m - qm) * S::RPP, real ? from + lo_step : V, real);
      }
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

template <int RP>
struct AdapterGradShape {
  static constexpr int RT = RP == 16 ? 16 : 32;               // ranks of a CTA
  static constexpr int MC = RP == 16 ? 128 : 64;              // columns of a CTA
  static constexpr int PP = MC * 2 + 16, TP = RT * 2 + 16;    // pitches of rows by columns and by rank
  static constexpr int STAGE = 16 * PP + 32 * TP;             // 16 rows: of the columns, of t's high and low parts
  static constexpr int STAGES = 2;                            // of a warp: what leaves room for two CTAs on an SM
  static constexpr int RING = 8 * STAGES * STAGE, PART = 8 * MC * RT * 4;
  static constexpr int BYTES = RING > PART ? RING : PART;     // (the warps' sums lie where the rows were)
};

// dA and dB: a CTA takes 64 or 128 columns of x or of dy and up to 32 ranks, and sums the products of those columns with u or t over the
// rows of all sequences that use its adapter. Its warps, and the CTAs of a cluster, take every so many blocks of 16 rows, each through a
// ring of its own, and wait for no other warp; their sums, those of warps that had a block, meet in one order. An adapter that nobody uses
// gets zeros. 16384 rows of 768 and 2304 columns, rank 16: 36 us (103 MB, 2.8 TB/s; with 64 columns, 128 bytes of a row, 40 us); rank
// 128: 110 us. 16 sequences of up to 27 rows, 33 adapters of rank 120, 6120 -> 200, all five kernels: 129 us (355 with the sums of all warps
// and two bytes a store).
template <typename T, int RP>
__global__ void __launch_bounds__(ADAPTER_THREADS, 2) adapter_grad_kernel(const __grid_constant__ AdapterGradParams p) {
  using S = AdapterGradShape<RP>;
  constexpr int MC = S::MC, RT = S::RT, MT = MC / 16, NT = RT / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  float* const part = reinterpret_cast<float*>(smem);  // (8, MC, RT), after the rows
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int a = blockIdx.y, rank0 = blockIdx.z * RT;
  const int k_tiles = p.da ? (p.K + MC - 1) / MC : 0;
  int c0 = (int)(blockIdx.x / cs);
  const bool of_a = c0 < k_tiles;
  c0 = (of_a ? c0 : c0 - k_tiles) * MC;
  const int C = of_a ? p.K : p.N;
  const T* const R = reinterpret_cast<const T*>(of_a ? p.x : p.dy);
  const int64_t sr = of_a ? p.x_sr : p.d_sr;
  const T* const W = reinterpret_cast<const T*>(of_a ? p.u : p.t);
  pdl_wait();
  pdl_launch_dependents();
  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;

  const uint32_t ring = smem_u32(smem) + warp * S::STAGES * S::STAGE;
  // a lane's pieces of a stage: rows pm, pm + PI, ... of the columns; rows tm (and tm + 8) of t's two parts
  constexpr int PI = 32 / (MC / 8);
  const int pm = lane / (MC / 8), pc = lane % (MC / 8) * 8, tm = lane / (RT / 8), tc = lane % (RT / 8) * 8;
  constexpr int TI = 32 / (RT / 8);
  const bool column = c0 + pc < C, ranks_here = rank0 + tc < p.r;
  const bool whole = c0 + MC <= C && rank0 + RT <= p.r;
  const int64_t step = PI * sr, lo_step = (int64_t)p.n_rows * p.r;
  int held = 0;                              // blocks asked for and not multiplied
  uint32_t put = ring, took = ring;          // where the next one goes, and the oldest lies
  const uint32_t row_to = pm * S::PP + pc * 2, t_to = 16 * S::PP + tm * S::TP + tc * 2;
  auto multiply = [&]() {
    const uint32_t ps = took, ts = ps + 16 * S::PP;
    took = took + S::STAGE == ring + S::STAGES * S::STAGE ? ring : took + S::STAGE;
    --held;
    uint32_t tb[2][NT / 2][4];
#pragma unroll
    for (int l = 0; l < 2; ++l)
#pragma unroll
      for (int n = 0; n < NT / 2; ++n) ldsm4t(tb[l][n], ts + (16 * l + (lane & 15)) * S::TP + (n * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t pa[4];  // the columns as the product's rows: 16 x 16 of the stage's rows (k) by columns (m), transposed
      ldsm4t(pa, ps + ((lane >> 4) * 8 + (lane & 7)) * S::PP + (m * 16 + ((lane >> 3) & 1) * 8) * 2);
#pragma unroll
      for (int l = 0; l < 2; ++l)
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          mma16<T>(acc[m][2 * n], pa, tb[l][n][0], tb[l][n][1]);
          mma16<T>(acc[m][2 * n + 1], pa, tb[l][n][2], tb[l][n][3]);
        }
    }
  };
  // one block is asked for; the one STAGES - 1 before it has arrived, and is multiplied
  auto ask = [&](int row0, int n) {  // 16 rows, n of them there
    __syncwarp();
    const uint32_t at = put;
    put = put + S::STAGE == ring + S::STAGES * S::STAGE ? ring : put + S::STAGE;
    const T* const from = R + (int64_t)(row0 + pm) * sr + c0 + pc;
    const T* const t = W + (int64_t)(row0 + tm) * p.r + rank0 + tc;
    if (whole && n >= 16) {
      const T* f = from;
#pragma unroll
      for (int q = 0; q < 16 / PI; ++q, f += step) cp16(at + row_to + PI * q * S::PP, f);
#pragma unroll
      for (int q = 0; q < 16 / TI; ++q) {
        cp16(at + t_to + TI * q * S::TP, t + TI * q * p.r);
        cp16(at + t_to + (16 + TI * q) * S::TP, t + TI * q * p.r + lo_step);
      }
    } else {
      for (int q = 0; q < 16 / PI; ++q) {
        const bool real = pm + PI * q < n && column;
        cp16(at + row_to + PI * q * S::PP, real ? from + q * step : R, real);
      }
      for (int q = 0; q < 16 / TI; ++q) {
        const bool real = tm + TI * q < n && ranks_here;
        cp16(at + t_to + TI * q * S::TP, real ? t + TI * q * p.r : W, real);
        cp16(at + t_to + (16 + TI * q) * S::TP, real ? t + TI * q * p.r + lo_step : W, real);
      }
    }
    cp_commit();
    if (++held >= S::STAGES) {
      cp_wait<S::STAGES - 1>();
      __syncwarp();
      multiply();
    }
  };
  int total = 0;  // the adapter's blocks
  {
    // this warp's blocks of 16 rows: every (8 cs)th of the adapter's, sequence after sequence
    const int turns = 8 * cs;
    int turn = rank * 8 + warp;  // blocks until the next one of this warp's
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + lane;
      int s0 = 0, s1 = 0;
      if (b < p.B && p.which[b] == a) {
        s0 = min(max(p.start[b], 0), p.n_rows);
        s1 = min(max(p.start[b + 1], 0), p.n_rows);
      }
      uint32_t some = __ballot_sync(0xffffffffu, s1 > s0);
      while (some) {
        const int from = __ffs(some) - 1;
        some &= some - 1;
        const int q0 = __shfl_sync(0xffffffffu, s0, from), q1 = __shfl_sync(0xffffffffu, s1, from);
        const int n = (q1 - q0 + 15) / 16;
        total += n;
        for (; turn < n; turn += turns) ask(q0 + turn * 16, q1 - q0 - turn * 16);
        turn -= n;
      }
    }
    cp_wait<0>();
    __syncwarp();
    while (held > 0) multiply();
  }
  const int ranks = min(RT, p.r - rank0);
  T* const da = reinterpret_cast<T*>(p.da) + ((int64_t)a * p.r + rank0) * p.K + c0;
  T* const db = reinterpret_cast<T*>(p.db) + ((int64_t)a * p.N + c0) * p.r + rank0;
  // eight elements of the outputs, dA as [r][K] and dB as [N][r]: the first's rank and column
  auto eight = [&](int e, int& c, int& m) {
    c = of_a ? e % RT : e % (RT / 8) * 8;
    m = of_a ? e / RT * 8 : e / (RT / 8);
    return c < ranks && c0 + m < C;
  };
  auto put8 = [&](int c, int m, const uint4& v) { *reinterpret_cast<uint4*>(of_a ? da + (int64_t)c * p.K + m : db + (int64_t)m * p.r + c) = v; };
  int c, m;
  if (total == 0) {  // (in all CTAs of a cluster)
    for (int e = rank * ADAPTER_THREADS + tid; e < MC * RT / 8; e += cs * ADAPTER_THREADS)
      if (eight(e, c, m)) put8(c, m, make_uint4(0u, 0u, 0u, 0u));
    return;
  }
  // the warps that had a block (one at least) have sums; they go where the rows were
  const int warps = max(1, min(8, total - rank * 8));
  __syncthreads();
  if (warp < warps) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* const to = part + (warp * MC + m * 16 + lane / 4) * RT + n * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(to) = make_float2(acc[m][n][0], acc[m][n][1]);
        *reinterpret_cast<float2*>(to + 8 * RT) = make_float2(acc[m][n][2], acc[m][n][3]);
      }
  }
  __syncthreads();
  if (cs == 1) {
    for (int e = tid; e < MC * RT / 8; e += ADAPTER_THREADS) {
      if (!eight(e, c, m)) continue;
      const int at = m * RT + c, by = of_a ? RT : 1;
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = part[at + i * by];
      for (int w = 1; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += part[w * MC * RT + at + i * by];
      put8(c, m, make_uint4(narrow2<T>(s[0], s[1]), narrow2<T>(s[2], s[3]), narrow2<T>(s[4], s[5]), narrow2<T>(s[6], s[7])));
    }
    return;
  }
  for (int e = tid; e < MC * RT; e += ADAPTER_THREADS) {
    float s = part[e];
#pragma unroll
    for (int w = 1; w < 8; ++w)
      if (w < warps) s += part[w * MC * RT + e];
    part[e] = s;
  }
  cluster_sync_all();
  // each CTA finishes a share of the columns
  const int m0 = MC * rank / cs, m1 = MC * (rank + 1) / cs, per = m1 - m0;
  for (int e = tid; e < per * ranks; e += ADAPTER_THREADS) {
    m = m0 + (of_a ? e % per : e / ranks);
    c = of_a ? e / per : e % ranks;
    float s = 0.f;
    for (int q = 0; q < cs; ++q) s += cluster_map(part, q)[m * RT + c];
    if (c0 + m < C) (of_a ? da[(int64_t)c * p.K + m] : db[(int64_t)m * p.r + c]) = from_f32<T>(s);
  }
  __syncwarp();
  cluster_sync_all();  // the others have read this CTA's part
}

}  // namespace ta
