// Attention over the 8-bit paged cache for many rows of one (sequence, kv head): prompt chunks and long runs of drafts, on
// the 5th-generation tensor cores. The mathematics and the cache are those of paged.cuh; here the products bound it.
//
// A CTA takes 128 rows (query-major: query i, head gq of the group -> row i * group + gq) and runs through 64-token blocks:
//   warps 4-7  converters: warp w reads the codes of one 16-token group (the next two blocks' are on their way to registers), turns
//              them into f16 and stores them as 128-byte-swizzled tiles: K (64 tokens x DH) and V transposed (DH x 64 tokens),
//              both K-major operands. A lane's fragment order gives it 32 bytes of a K row and token pairs of V columns, so
//              neither store meets a bank twice.
//   warp 8     one thread issues tcgen05.mma: S = Q K^T of block j, then O += P V of block j - 1 (accumulator in tensor
//              memory), so that the softmax of one block runs beside the products of its neighbours.
//   warps 0-3  softmax, one thread per row: maximum, weights (f16, into shared memory), denominator; O is rescaled in tensor
//              memory only when a row's reference has to rise by more than 2^8.
// The open page is the last block: 16-bit elements as they are, with a copy of the queries in that type (its infinities and NaN
// join at the end, row by row).
// What bounds it is the chain of latencies of a block's softmax step (scores out of tensor memory, maximum, weights, their way
// through shared memory to the next product): without the exponentials, the stores or the conversions it is 1 to 4 % faster.
// Two sequences of up to 4000 tokens, chunks of 512, 12 heads of 64: 41 us; 16 sequences of 8000, 40 rows for each of 4 heads:
// 59 us at head dim 64, 92 at 128 (one CTA an SM). Where the tiles do not fill the GPU, the blocks of a tile are shared by several
// CTAs; their states meet in the workspace and the last to come (a counter per tile) joins them.
#pragma once
#include <cstddef>
#include "paged.cuh"
#include "tc.cuh"

namespace ta {

constexpr int TILE_ROWS = 128;
constexpr int TILE_KT = 64;
constexpr int TILE_THREADS = 288;
constexpr int TILE_MAX_SPLITS = 8;
constexpr int K_PAGED_TILE = 19;

template <typename T, int DH>
struct TileShape {
  static constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int NS = 2;                          // K and V stages (as many as score and weight buffers)
  static constexpr int HALVES = DH / 64;                // 64-dim column blocks of Q and K
  static constexpr int Q_BYTES = TILE_ROWS * DH * 2;
  static constexpr int K_BYTES = TILE_KT * DH * 2;      // and of V
  static constexpr int P_BYTES = TILE_ROWS * TILE_KT * 2;
  static constexpr int Q2 = BF ? Q_BYTES : 0;           // the queries in bf16, for the open page
  static constexpr int BYTES = Q_BYTES + Q2 + NS * 2 * K_BYTES + 2 * P_BYTES;
  static constexpr int CTAS = DH == 64 ? 2 : 1;         // per SM
  static constexpr int STATE = TILE_ROWS * (DH + 2);    // floats: numerators (4 dims of every row together), maxima, sums
};

struct TileBars {
  uint64_t k_full[2], v_full[2], s_full[2], s_free[2], p_full[2], o_full[2], mma_done;
  // per block (of four in turn) and 16-token group: key scale, log2 of the value scale, its inverse
  alignas(16) float scale[4][4][4];
  uint32_t tmem_base;
  int abort_flag, last;
  int odd;  // the open page holds an infinity or NaN among its values
};

static_assert(offsetof(TileBars, scale) % 16 == 0, "the scales are read as float4");

struct TileParams {
  AttnParams a;
  int tiles, splits;
  int32_t* counters;  // (B, Hkv, tiles), zero between launches
  float* states;      // (B, Hkv, tiles, splits) states
};

// 16 consecutive fp32 columns of this thread's TMEM lane on their way to v; complete after tmem_got.
__device__ __forceinline__ void tmem_get16(uint32_t taddr, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_got(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));  // no use of v moves above the wait
}

// A bounded wait for a phase that is usually complete already, or about to be: tests without suspending, and looks at the
// clock (itself hundreds of cycles) only after some time. With the waits that suspend and read it first a softmax step spent
// 700 of 3600 cycles on barriers that were already complete.
__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t parity, int where) {
  uint64_t t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((spins & 255u) == 255u) {
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > TA_WAIT_LIMIT_NS) {
        record_error(DEV_WAIT_TIMEOUT, K_PAGED_TILE, where, (int)parity);
        return false;
      }
    }
  }
}

// Two fp32 at a time, and the largest of three.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f32x2_parts(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma_x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// a 16-byte piece of a swizzled tile's row (128 bytes)
__device__ __forceinline__ unsigned char* tile_piece(unsigned char* tile, int row, int c) {
  return tile + row * 128 + ((c ^ (row & 7)) << 4);
}

template <typename T, int DH, bool PROBE = false>
__global__ void __launch_bounds__(TILE_THREADS, TileShape<T, DH>::CTAS) paged_tile_kernel(TileParams tp) {
  using C = TileShape<T, DH>;
  using S = PageShape<DH>;
  constexpr int NS = C::NS;
  constexpr float SHIFT = 6.f, RISE = 8.f;  // weights stay below 2^(SHIFT + RISE) = 2^14
  constexpr uint32_t TM_S = 0, TM_O = 128, TM_COLS = 256;
  const AttnParams& p = tp.a;
  extern __shared__ unsigned char tile_smem_raw[];
  const uint32_t raw_a = smem_u32(tile_smem_raw);
  unsigned char* sQ = tile_smem_raw + (((raw_a + 1023u) & ~1023u) - raw_a);
  unsigned char* sQ2 = C::BF ? sQ + C::Q_BYTES : sQ;
  unsigned char* sKV = sQ + C::Q_BYTES + C::Q2;
  unsigned char* sP = sKV + NS * 2 * C::K_BYTES;
  TileBars& bar = *reinterpret_cast<TileBars*>(sP + 2 * C::P_BYTES);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % tp.splits, tile = tp.tiles - 1 - (int)(blockIdx.x / tp.splits);  // heavy (late) tiles first
  const int b = blockIdx.z, h = blockIdx.y, row0 = tile * TILE_ROWS;
  pdl_wait();
  pdl_launch_dependents();
  NewRows nr;
  if (!new_rows(p.start, p.pos, b, p.n_rows, p.max_new, p.c, K_PAGED_ATTN, nr)) return;
  const int group = p.Hq / p.c.Hkv, R = nr.n * group, P = p.c.P, lp = 31 - __clz(P);
  if (row0 >= R) return;
  const int len = nr.pos + nr.n, n_full = len >> lp;
  const int qlo = nr.pos + row0 / group, qhi = nr.pos + (min(R, row0 + TILE_ROWS) - 1) / group;
  const int p0 = (p.window > 0 ? max(0, qlo - p.window + 1) : 0) >> lp, p1 = min(n_full, (qhi >> lp) + 1);
  const int first_tok = p0 << lp, limit = p1 << lp;
  const int n_code = (limit - first_tok + TILE_KT - 1) / TILE_KT;              // blocks of full pages
  const int n_all = n_code + ((n_full << lp) <= qhi ? 1 : 0);                  // and the open page
  const int j0 = (int)((int64_t)n_all * split / tp.splits), j1 = (int)((int64_t)n_all * (split + 1) / tp.splits);
  const int nblk = j1 - j0;

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar.k_full[s], 4);
      mbar_init(&bar.v_full[s], 4);
      mbar_init(&bar.s_full[s], 1);
      mbar_init(&bar.s_free[s], 4);
      mbar_init(&bar.p_full[s], 4);
      mbar_init(&bar.o_full[s], 1);
    }
    mbar_init(&bar.mma_done, 1);
    bar.abort_flag = bar.odd = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&bar.tmem_base, TM_COLS);
    tmem_relinquish();
  }
  // ---- the queries: a thread a row
  const int rr = row0 + tid;
  float cs = 1.f;
  int qpos = -1;
  if (warp < 4) {
    uint4 q[DH / 8];
    const bool live = rr < R;
    const T* src = reinterpret_cast<const T*>(p.q);
    if (live) {
      src += (int64_t)(nr.row0 + rr / group) * p.q_sr + (int64_t)(h * group + rr % group) * p.q_sh;
      qpos = nr.pos + rr / group;
    }
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < DH / 8; ++c) q[c] = live ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int c = 0; c < DH / 8; ++c) {
      float x[8];
      load_vec_f32<T>(reinterpret_cast<const T*>(&q[c]), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
    }
    // as in RowTile: the row's power of two, the sign of the scale, a zero row at scale 0
    const int ex = min(7 + 127 - (int)(__float_as_uint(top) >> 23), 120);
    const float up = p.scale == 0.f ? 0.f : copysignf(__int_as_float((ex + 127) << 23), p.scale);
    cs = p.scale == 0.f ? 1.f : fabsf(p.scale) * 1.4426950408889634f * __int_as_float((127 - ex) << 23);
#pragma unroll
    for (int c = 0; c < DH / 8; ++c) {
      float x[8];
      load_vec_f32<T>(reinterpret_cast<const T*>(&q[c]), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= up;
      const int at = (c >> 3) * TILE_ROWS * 128;
      store_vec_from_f32<__half>(reinterpret_cast<__half*>(tile_piece(sQ + at, tid, c & 7)), x);
      if constexpr (C::BF) store_vec_from_f32<T>(reinterpret_cast<T*>(tile_piece(sQ2 + at, tid, c & 7)), x);
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp >= 4 && warp < 8) {
    // ---------------------------------------------------------------- converters
    const int cw = warp - 4;
    constexpr int KW = S::HG * 2 * (S::E / 4), VW = S::C * 2 * S::M;  // words of a lane: keys, values
    const int32_t* table = p.c.table + b * p.c.table_sb;
    const int rec = 2 * P * DH + 16;
    const int n_mine = min(j1, n_code) - j0;  // blocks of codes
    auto entry = [&](int j) {
      const int page = min(p0 + ((j * TILE_KT + cw * 16) >> lp), p1 - 1);  // beyond the last page: the last again (masked)
      return table[page];
    };
    auto fetch = [&](int j, int phys, uint32_t (&kw)[KW], uint32_t (&vw)[VW], float4& sc) {
      const unsigned char* r = record_of(p.c, phys, h, rec, b);
      const unsigned char* k = r + ((j * TILE_KT + cw * 16) & (P - 1)) * DH;
      const unsigned char* v = k + P * DH;
#pragma unroll
      for (int x = 0; x < KW / 4; ++x) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(k) + x * 32 + lane);
        kw[4 * x] = w.x; kw[4 * x + 1] = w.y; kw[4 * x + 2] = w.z; kw[4 * x + 3] = w.w;
      }
#pragma unroll
      for (int x = 0; x < VW / 4; ++x) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(v) + x * 32 + lane);
        vw[4 * x] = w.x; vw[4 * x + 1] = w.y; vw[4 * x + 2] = w.z; vw[4 * x + 3] = w.w;
      }
      sc = __ldg(reinterpret_cast<const float4*>(r + 2 * P * DH));
    };
    // block n: its codes are in the registers given, which then take those of block n + 2 (two sets in turn: moving one to
    // the other would wait for the loads); ent: the table entry of that block
    bool ok = true;
    auto block = [&](int n, uint32_t (&kw)[KW], uint32_t (&vw)[VW], float4& sc, int& ent) -> bool {
      const int st = n % NS;
      unsigned char* sK = sKV + st * 2 * C::K_BYTES;
      unsigned char* sV = sK + C::K_BYTES;
      // K's stage is free when the scores of block n - 2 are there, long before V's (the products of block n - 2 with the
      // weights): so K goes first, and the next scores do not wait for the softmax. (The scales' place was last read by the
      // softmax of block n - 4, which V's stage of block n - 1 waited for.)
      auto free_of = [&](uint64_t* done, int where) {
        if (n >= NS && !mbar_wait_bounded(done + st, ((n / NS) - 1) & 1, K_PAGED_TILE, where)) {
          atomicExch(&bar.abort_flag, 1);
          ok = false;
        }
        if (*reinterpret_cast<volatile int*>(&bar.abort_flag)) ok = false;
        return ok;
      };
      auto filled = [&](uint64_t* full) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full + st);
      };
      if (!free_of(bar.s_full, 1)) return false;
      const int row = cw * 16 + g;  // a K row of this lane, and the one 8 further on
      if (n < n_mine) {
#pragma unroll
        for (int hg = 0; hg < S::HG; ++hg)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t f[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) codes_f16x4(kw[(hg * 2 + r) * 4 + e], f[2 * e], f[2 * e + 1]);
            unsigned char* tileK = sK + hg * TILE_KT * 128;
            *reinterpret_cast<uint4*>(tile_piece(tileK, row + 8 * r, 2 * t)) = make_uint4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<uint4*>(tile_piece(tileK, row + 8 * r, 2 * t + 1)) = make_uint4(f[4], f[5], f[6], f[7]);
          }
        float lv, iv;
        value_factors(sc, lv, iv);
        if (lane == 0) *reinterpret_cast<float4*>(bar.scale[n & 3][cw]) = make_float4(sc.x, lv, iv, 0.f);
        filled(bar.k_full);
        if (!free_of(bar.o_full, 11)) return false;
#pragma unroll
        for (int x = 0; x < VW; ++x) {  // (c, m, r): 4 tokens of one dim
          const int d = (x / 2) * 16 + (x & 1) * 8 + g;
          uint32_t lo, hi;
          codes_f16x4(vw[x], lo, hi);
          *reinterpret_cast<uint32_t*>(tile_piece(sV, d, 2 * cw) + 4 * t) = lo;
          *reinterpret_cast<uint32_t*>(tile_piece(sV, d, 2 * cw + 1) + 4 * t) = hi;
        }
      } else {
        // the open page: 16-bit elements; rows it does not hold are zeroed (their keys are masked as well)
        const T* tk = reinterpret_cast<const T*>(p.c.tail) +
                      ((((int64_t)b * p.c.Hkv + h) * 2 + (n_full & 1)) * 2) * ((int64_t)P * DH) + cw * 16 * DH;
        const T* tv = tk + (int64_t)P * DH;
        const int held = len - (n_full << lp) - cw * 16;  // tokens of this group
        if (held > 0) {
#pragma unroll
          for (int hg = 0; hg < S::HG; ++hg)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              uint32_t w[8];
              load_words<32>(tk + ((hg * 2 + r) * 32 + lane) * S::E, w);
              unsigned char* tileK = sK + hg * TILE_KT * 128;
              *reinterpret_cast<uint4*>(tile_piece(tileK, row + 8 * r, 2 * t)) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(tile_piece(tileK, row + 8 * r, 2 * t + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
        if (lane == 0) *reinterpret_cast<float4*>(bar.scale[n & 3][cw]) = make_float4(1.f, 0.f, 1.f, 0.f);
        filled(bar.k_full);
        if (!free_of(bar.o_full, 11)) return false;
        const uint32_t keep0 = (2 * t < held ? 0xffffu : 0u) | (2 * t + 1 < held ? 0xffff0000u : 0u);
        const uint32_t keep1 = (2 * t + 8 < held ? 0xffffu : 0u) | (2 * t + 9 < held ? 0xffff0000u : 0u);
        uint32_t odd = 0u;
#pragma unroll 4  // (once a CTA: unrolled whole, the code around it took 42.5 us for the chunk of 512, so 41.1)
        for (int x = 0; x < VW; ++x) {
          const int d = (x / 2) * 16 + (x & 1) * 8 + g;
          uint32_t w[2] = {0u, 0u};
          if (held > 0) load_words<8>(tv + ((x / (2 * S::M)) * 32 + lane) * 8 * S::M + (x % (2 * S::M)) * 4, w);
          w[0] &= keep0;
          w[1] &= keep1;
          odd |= odd2<T>(w[0]) | odd2<T>(w[1]);
          *reinterpret_cast<uint32_t*>(tile_piece(sV, d, 2 * cw) + 4 * t) = finite2<T>(w[0]);
          *reinterpret_cast<uint32_t*>(tile_piece(sV, d, 2 * cw + 1) + 4 * t) = finite2<T>(w[1]);
        }
        if (odd) bar.odd = 1;
      }
      if (n + 2 < n_mine) {
        fetch(j0 + n + 2, ent, kw, vw, sc);
        if (n + 4 < n_mine) ent = entry(j0 + n + 4);
      }
      filled(bar.v_full);
      return true;
    };
    uint32_t ka[KW], va[VW], kb[KW], vb[VW];
    float4 sa, sb;
    int ea = 0, eb = 0;
    if (n_mine > 0) ea = entry(j0);
    if (n_mine > 1) eb = entry(j0 + 1);
    if (n_mine > 0) fetch(j0, ea, ka, va, sa);
    if (n_mine > 1) fetch(j0 + 1, eb, kb, vb, sb);
    if (n_mine > 2) ea = entry(j0 + 2);
    if (n_mine > 3) eb = entry(j0 + 3);
    const bool absent = PROBE && (int)blockIdx.x == p.probe && blockIdx.y + blockIdx.z == 0;  // its tiles never come
    for (int n = 0; n < nblk && !absent; n += 2) {
      if (!block(n, ka, va, sa, ea)) break;
      if (n + 1 < nblk && !block(n + 1, kb, vb, sb, eb)) break;
    }
  } else if (warp == 8) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0 && nblk > 0) {
      constexpr uint32_t S_F16 = umma_idesc_f16(TILE_ROWS, TILE_KT, false, false), S_T = umma_idesc_f16(TILE_ROWS, TILE_KT, C::BF, false);
      constexpr uint32_t O_F16 = umma_idesc_f16(TILE_ROWS, DH, false, false), O_T = umma_idesc_f16(TILE_ROWS, DH, C::BF, false);
      const uint32_t tS = bar.tmem_base + TM_S, tO = bar.tmem_base + TM_O;
      const uint32_t aQ = smem_u32(sQ), aQ2 = smem_u32(sQ2), aKV = smem_u32(sKV), aP = smem_u32(sP);
      bool ok = true;
      auto issue_pv = [&](int n) -> bool {
        if (!tile_wait(&bar.v_full[n % NS], (n / NS) & 1, 12) ||
            !tile_wait(&bar.p_full[n & 1], (n >> 1) & 1, 2))
          return false;
        if (*reinterpret_cast<volatile int*>(&bar.abort_flag)) return false;
        tc_fence_after();
        const uint32_t pa = aP + (n & 1) * C::P_BYTES, va = aKV + (n % NS) * 2 * C::K_BYTES + C::K_BYTES;
#pragma unroll
        for (int k = 0; k < TILE_KT / 16; ++k)
          umma_f16(tO, sw128_desc(pa + k * 32, 16, 1024), sw128_desc(va + k * 32, 16, 1024), j0 + n < n_code ? O_F16 : O_T,
                   n > 0 || k > 0);
        umma_commit(&bar.o_full[n & 1]);
        return true;
      };
      for (int n = 0; n < nblk; ++n) {
        if (!(ok = tile_wait(&bar.k_full[n % NS], (n / NS) & 1, 3))) break;
        if (n >= 2 && !(ok = tile_wait(&bar.s_free[n & 1], ((n >> 1) - 1) & 1, 4))) break;
        if (*reinterpret_cast<volatile int*>(&bar.abort_flag)) { ok = false; break; }
        tc_fence_after();
        const bool code = j0 + n < n_code;
        const uint32_t qa = code ? aQ : aQ2, ka = aKV + (n % NS) * 2 * C::K_BYTES;
#pragma unroll
        for (int k = 0; k < DH / 16; ++k)
          umma_f16(tS + (n & 1) * TILE_KT, sw128_desc(qa + (k >> 2) * (TILE_ROWS * 128) + (k & 3) * 32, 16, 1024),
                   sw128_desc(ka + (k >> 2) * (TILE_KT * 128) + (k & 3) * 32, 16, 1024), code ? S_F16 : S_T, k > 0);
        umma_commit(&bar.s_full[n & 1]);
        if (n >= 1 && !(ok = issue_pv(n - 1))) break;
      }
      if (ok) ok = issue_pv(nblk - 1);
      if (!ok) atomicExch(&bar.abort_flag, 1);
      umma_commit(&bar.mma_done);
      mbar_wait_bounded(&bar.mma_done, 0, K_PAGED_TILE, 5);  // every MMA of this CTA has completed
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax (thread = row)
    const uint32_t lane_base = bar.tmem_base + ((uint32_t)(warp * 32) << 16);
    float ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int n = 0; n < nblk; ++n) {
      // The scores of block n: the issuing thread had seen its K (and scales) complete, and the same arrival stands for every
      // product issued before, those of block n - 2 with the weights among them, whose buffer this step overwrites.
      if (!tile_wait(&bar.s_full[n & 1], (n >> 1) & 1, 7)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool code = j0 + n < n_code;
      const int tok0 = code ? first_tok + (j0 + n) * TILE_KT : n_full << lp;
      const int lim = code ? limit : len;
      const bool mask = tok0 + TILE_KT - 1 > min(qlo, lim - 1) || (p.window > 0 && tok0 <= qhi - p.window);
      // this row's visible columns are [c0, c1)
      const int c1 = min(min(qpos + 1, lim) - tok0, TILE_KT), c0 = p.window > 0 ? qpos - p.window + 1 - tok0 : 0;
      float ks[4], lv[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 f = *reinterpret_cast<const float2*>(bar.scale[n & 3][x]);
        ks[x] = f.x * cs;
        lv[x] = f.y;
      }
      // two passes over the scores, 16 columns at a time with the next ones on their way: all 64 at once do not fit the 96
      // registers that two CTAs an SM leave a thread
      const uint32_t tS = lane_base + TM_S + (n & 1) * TILE_KT;
      float va[16], vb[16];
      tmem_get16(tS, va);
      tmem_got(va);
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float(&v)[16] = x & 1 ? vb : va;
        float(&next)[16] = x & 1 ? va : vb;
        if (x < 3) tmem_get16(tS + (x + 1) * 16, next);
        if (mask) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (x * 16 + i < c0 || x * 16 + i >= c1) v[i] = -INFINITY;
        }
        float m0 = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
        m0 = max3(m0, v[6], v[7]);
        m1 = max3(m1, v[8], v[9]);
        m0 = max3(m0, v[10], v[11]);
        m1 = max3(m1, v[12], v[13]);
        m0 = max3(m0, v[14], v[15]);
        top = fmaxf(top, fmaf(fmaxf(m0, m1), ks[x], lv[x]));
        if (x < 3) tmem_got(next);
      }
      tmem_get16(tS, va);
      const bool rise = top > ref + RISE || (ref == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, rise)) {
        const float f = rise && ref != -INFINITY ? exp2_fast(ref - top) : 1.f;
        if (rise) ref = top;
        l *= f;
        if (n > 0) {
          // O holds the blocks before this one: their products have to be complete
          if (!tile_wait(&bar.o_full[(n - 1) & 1], ((n - 1) >> 1) & 1, 8)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DH; c += 32) {
            float o[32];
            tmem_ld32(lane_base + TM_O + c, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= f;
            tmem_st32(lane_base + TM_O + c, o);
          }
          tmem_wait_st();
        }
      }
      const float base = (ref == -INFINITY ? 0.f : ref) - SHIFT;
      unsigned char* tileP = sP + (n & 1) * C::P_BYTES;
      tmem_got(va);
      auto weights = [&](auto masked, auto type) {
        using W = decltype(type);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float(&w)[16] = x & 1 ? vb : va;
          float(&next)[16] = x & 1 ? va : vb;
          if (x < 3) tmem_get16(tS + (x + 1) * 16, next);
          const uint64_t k2 = f32x2(ks[x], ks[x]), b2 = f32x2(lv[x] - base, lv[x] - base);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 e = f32x2_parts(fma_x2(f32x2(w[i], w[i + 1]), k2, b2));
            w[i] = exp2_fast(e.x);
            w[i + 1] = exp2_fast(e.y);
          }
          if constexpr (decltype(masked)::value) {  // a masked token weighs 0 whatever its score and scales are
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (x * 16 + i < c0 || x * 16 + i >= c1) w[i] = 0.f;
          }
          uint64_t a0 = f32x2(w[0], w[1]), a1 = f32x2(w[2], w[3]);
#pragma unroll
          for (int i = 4; i < 16; i += 4) {
            a0 = add_x2(a0, f32x2(w[i], w[i + 1]));
            a1 = add_x2(a1, f32x2(w[i + 2], w[i + 3]));
          }
          const float2 a = f32x2_parts(add_x2(a0, a1));
          const float sum = a.x + a.y;
          l += sum == 0.f ? 0.f : sum * bar.scale[n & 3][x][2];
          store_vec_from_f32<W>(reinterpret_cast<W*>(tile_piece(tileP, tid, 2 * x)), w);
          store_vec_from_f32<W>(reinterpret_cast<W*>(tile_piece(tileP, tid, 2 * x + 1)), w + 8);
          if (x < 3) tmem_got(next);
        }
      };
      if (!mask)
        weights(std::false_type{}, __half{});
      else if (code)
        weights(std::true_type{}, __half{});
      else
        weights(std::true_type{}, T{});  // (the open page is never seen whole)
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar.s_free[n & 1]);
        mbar_arrive(&bar.p_full[n & 1]);
      }
    }
    if (ok && nblk > 0) ok = tile_wait(&bar.o_full[(nblk - 1) & 1], ((nblk - 1) >> 1) & 1, 10);
    if (!ok) atomicExch(&bar.abort_flag, 1);
    tc_fence_after();
    named_bar_sync(1, 128);
    const bool good = *reinterpret_cast<volatile int*>(&bar.abort_flag) == 0;  // one outcome for the 4 warps
    named_bar_sync(1, 128);
    const bool live = rr < R;
    T* out = nullptr;
    int64_t out_row = 0;
    int hq = 0;
    if (live) {
      out_row = nr.row0 + rr / group;
      hq = h * group + rr % group;
      out = reinterpret_cast<T*>(p.out) + out_row * p.o_sr + (int64_t)hq * p.o_sh;
    }
    auto finish = [&](int odd) {
      if (__builtin_expect(odd != 0, 0) && live)
        add_odd<T, DH>(open_values<T, DH>(p.c, b, h, n_full), n_full << lp, p.window > 0 ? qpos - p.window + 1 : 0, qpos + 1, 0, DH,
                       1, out);
      if (p.lse && live) p.lse[out_row * p.Hq + hq] = l == 0.f ? -INFINITY : (ref - SHIFT + log2f(l)) * 0.69314718055994531f;
    };
    if (!good) {  // a wait that gave up: the rows are NaN, and the tile's counter comes back to zero all the same
      l = NAN;
      ref = -INFINITY;
    }
    if (tp.splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < DH; c += 32) {
        float o[32];
        if (good) tmem_ld32(lane_base + TM_O + c, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = good ? o[i] * inv : NAN;
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) store_vec_from_f32<T>(out + c + i, o + i);
        }
      }
      finish(*reinterpret_cast<volatile int*>(&bar.odd));
    } else {
      // this CTA's share of the blocks; the last of the tile's CTAs joins them in order
      const int64_t item = ((int64_t)b * p.c.Hkv + h) * tp.tiles + tile;
      float* states = tp.states + item * tp.splits * C::STATE;
      float* mine = states + split * C::STATE;
      const bool have = good && nblk > 0;
#pragma unroll 1
      for (int c = 0; c < DH; c += 32) {
        float o[32];
        if (have) tmem_ld32(lane_base + TM_O + c, o);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          __stcg(reinterpret_cast<float4*>(mine) + (c + i) / 4 * TILE_ROWS + tid,
                 have ? make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]) : make_float4(0.f, 0.f, 0.f, 0.f));
      }
      __stcg(mine + TILE_ROWS * DH + tid, ref);
      __stcg(mine + TILE_ROWS * (DH + 1) + tid, l);
      __threadfence();
      named_bar_sync(1, 128);
      if (tid == 0) {  // arrivals, and above them those of odd shares
        const int before = atomicAdd(tp.counters + item, 1 + (bar.odd << 16));
        bar.last = (before & 0xffff) == tp.splits - 1;
        bar.odd |= before >> 16;
      }
      named_bar_sync(1, 128);
      if (bar.last) {
        __threadfence();
        if (tid == 0) tp.counters[item] = 0;
        float f[TILE_MAX_SPLITS];
        ref = -INFINITY;
#pragma unroll
        for (int s = 0; s < TILE_MAX_SPLITS; ++s) {
          f[s] = -INFINITY;
          if (s < tp.splits) f[s] = __ldcg(states + s * C::STATE + TILE_ROWS * DH + tid);
          ref = fmaxf(ref, f[s]);
        }
        l = 0.f;
#pragma unroll
        for (int s = 0; s < TILE_MAX_SPLITS; ++s) {
          // (a share that saw nothing, or nothing but NaN, has no maximum: its sums count as they are)
          f[s] = s >= tp.splits ? 0.f : (f[s] == -INFINITY ? 1.f : exp2_fast(f[s] - ref));
          if (s < tp.splits) l += __ldcg(states + s * C::STATE + TILE_ROWS * (DH + 1) + tid) * f[s];
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int c = 0; c < DH; c += 8) {
          float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < TILE_MAX_SPLITS; ++s)
            if (s < tp.splits) {
              const float4* src = reinterpret_cast<const float4*>(states + s * C::STATE) + c / 4 * TILE_ROWS + tid;
              const float4 x = __ldcg(src), y = __ldcg(src + TILE_ROWS);
              o[0] += x.x * f[s]; o[1] += x.y * f[s]; o[2] += x.z * f[s]; o[3] += x.w * f[s];
              o[4] += y.x * f[s]; o[5] += y.y * f[s]; o[6] += y.z * f[s]; o[7] += y.w * f[s];
            }
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= inv;
          if (live) store_vec_from_f32<T>(out + c, o);
        }
        finish(*reinterpret_cast<volatile int*>(&bar.odd));
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(bar.tmem_base, TM_COLS);
  }
}

}  // namespace ta
