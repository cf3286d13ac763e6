// Verification of drafted tokens (speculative sampling): the drafts that stand and the token that follows them, from the
// target's and the draft's probabilities and given uniform numbers.
//   draft i stands while u_i q_i(d_i) < p_i(d_i);  a = the drafts that stand before the first that does not (at most n)
//   the next token is drawn from max(p_a - q_a, 0), or from p_a when every draft stood or nothing is left of it, by the
//   inverse of its cumulative sum at u_G (a number of its own: u_a is not uniform any more once draft a has failed).
// The weights are summed in fixed point (steps of 2^-38, 64-bit integers; uniform numbers as 24 bits): the sums do not
// depend on their order, so the token is the same for every split of the vocabulary.
#pragma once
#include "common.cuh"

namespace ta {

// A cluster of CTAs takes a sequence: each CTA finds where the drafts stop (a handful of loads), then sums its share of the row
// that the token comes from; the shares meet through distributed shared memory, and the CTA whose share holds the mark
// looks through the one warp-sized piece that does. Latency-bound: two dependent loads, one pass over the row, one cluster
// barrier, one more look at a piece (in L2). Vocabulary 50304, four drafts, fp32: one sequence 7.6 us, 64 sequences 13 us (26 MB of
// rows at most); 256 of 32000, eight drafts, bf16: 18 us
// (all CTAs resident at once; the second look is at a whole warp's 2048 words).
constexpr int VERIFY_THREADS = 256;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int VERIFY_MAX_CLUSTER = 8;

struct VerifyParams {
  const void *p, *q;
  int64_t p_sb, p_sr, q_sb, q_sr;
  const int64_t* drafts;  // (B, G)
  const float* u;         // (B, G + 1): one for each draft, the last for the draw
  const int32_t* n;       // (B,) drafts of each sequence, or null (G)
  int B, G, V;
  int seg;                // words of a warp: a multiple of 32 16-byte pieces
  int64_t* tokens;        // (B, G + 1)
  int32_t* accepted;      // (B,)
};

// max(p - q, 0) in steps of 2^-38, rounded down; what is not a number weighs nothing. (By way of 32 bits: a product of 2^31
// or more is a multiple of 2^8.)
__device__ __forceinline__ unsigned long long left_over(float p, float q) {
  const float d = p > q ? fminf(__fsub_rn(p, q), 1.f) : 0.f;
  const bool big = d >= 0.0078125f;
  const uint32_t i = __float2uint_rz(d * (big ? 1073741824.f : 274877906944.f));
  return big ? (unsigned long long)i << 8 : (unsigned long long)i;
}

template <typename T>
__global__ void __launch_bounds__(VERIFY_THREADS, 4) verify_kernel(VerifyParams a) {
  constexpr int VEC = TypeInfo<T>::VEC;
  __shared__ int s_acc;
  __shared__ unsigned long long s_sum[VERIFY_WARPS];
  __shared__ unsigned long long s_total[2];  // of this CTA: with the draft's row taken off, and without
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int b = blockIdx.x / cs;
  const T* P = reinterpret_cast<const T*>(a.p) + b * a.p_sb;
  const T* Q = reinterpret_cast<const T*>(a.q) + b * a.q_sb;
  if (tid == 0) s_acc = 0x7fffffff;
  pdl_wait();
  pdl_launch_dependents();
  const float uf = a.u[(int64_t)b * (a.G + 1) + a.G];
  int n = a.n ? a.n[b] : a.G;
  __syncthreads();
  // (drafts beyond n are read with the others, and do not count)
  for (int i = tid; i < a.G; i += VERIFY_THREADS) {
    const int64_t d = a.drafts[(int64_t)b * a.G + i];
    const float ui = a.u[(int64_t)b * (a.G + 1) + i];
    bool ok = false;
    if (d >= 0 && d < a.V)
      ok = __fmul_rn(ui, to_f32(Q[i * a.q_sr + d])) < to_f32(P[i * a.p_sr + d]);
    else if (i < n)
      record_error(DEV_INDEX_RANGE, K_VERIFY, b, (int)d);
    if (!ok) atomicMin(&s_acc, i);
  }
  if (n < 0 || n > a.G) {
    if (tid == 0) record_error(DEV_INDEX_RANGE, K_VERIFY, b, n);
    n = n < 0 ? 0 : a.G;
  }
  __syncthreads();
  const int acc = min(s_acc, n);
  const T* pr = P + acc * a.p_sr;
  bool rest = acc < n;  // whether the draft's row is taken off
  const T* qr = rest ? Q + acc * a.q_sr : pr;
  const bool vec = ((reinterpret_cast<uintptr_t>(pr) | reinterpret_cast<uintptr_t>(qr)) & 15u) == 0;
  // the weights of the VEC words from v on (0 beyond the row)
  auto weights = [&](int v, unsigned long long (&w)[VEC]) {
    if (vec && v + VEC <= a.V) {
      float x[VEC], y[VEC];
      ldg_vec_f32<T>(pr + v, x);
      if (rest) ldg_vec_f32<T>(qr + v, y);
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = left_over(x[e], rest ? y[e] : 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        w[e] = v + e < a.V ? left_over(to_f32(pr[v + e]), rest ? to_f32(qr[v + e]) : 0.f) : 0ull;
    }
  };
  const int v0 = (rank * VERIFY_WARPS + warp) * a.seg, v1 = min(a.V, v0 + a.seg);
  unsigned long long total = 0, before = 0, own = 0;
  for (int pass = 0; pass < 2; ++pass) {
    unsigned long long sum = 0;
    int v = v0 + lane * VEC;
    if (vec) {
      // 4 pieces of each row in flight per lane
      constexpr int U = 4;
      for (; v + VEC <= v1; v += U * 32 * VEC) {
        uint4 x[U], y[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          x[i] = y[i] = make_uint4(0u, 0u, 0u, 0u);
          if (v + i * 32 * VEC + VEC <= v1) {
            x[i] = __ldg(reinterpret_cast<const uint4*>(pr + v + i * 32 * VEC));
            if (rest) y[i] = __ldg(reinterpret_cast<const uint4*>(qr + v + i * 32 * VEC));
          }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          float fx[VEC], fy[VEC];
          load_vec_f32<T>(reinterpret_cast<const T*>(&x[i]), fx);
          load_vec_f32<T>(reinterpret_cast<const T*>(&y[i]), fy);
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum += left_over(fx[e], fy[e]);
        }
      }
      // the piece that the row ends in: the first that the loop left out, of one lane
      const int cut = v1 / VEC * VEC;
      v = cut < v1 && cut >= v0 && ((cut - v0) / VEC & 31) == lane ? cut : v1;
    }
    for (; v < v1; v += 32 * VEC) {
      unsigned long long w[VEC];
      weights(v, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += w[e];
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      unsigned long long x = lane < VERIFY_WARPS ? s_sum[lane] : 0ull;
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (lane == 0) s_total[pass] = x;
    }
    cluster_sync_all();
    total = before = 0;
    for (int r = 0; r < cs; ++r) {
      const unsigned long long x = *cluster_map(&s_total[pass], r);
      if (r == rank) {
        before = total;
        own = x;
      }
      total += x;
    }
    // nothing left over: the target's row itself (every CTA of the cluster sees the same total)
    if (total > 0 || !rest) break;
    rest = false;
  }
  cluster_arrive();  // this CTA has read the others' totals
  const unsigned long long u24 = uf > 0.f ? (unsigned long long)fminf(uf * 16777216.f, 16777215.f) : 0ull;
  const unsigned long long mark = (total >> 24) * u24 + (((total & 0xffffffull) * u24) >> 24);
  const bool mine = total > 0 ? mark >= before && mark < before + own : rank == 0;
  if (mine && warp == 0) {
    int64_t tok = a.V - 1;
    if (total > 0) {
      const unsigned long long x = lane < VERIFY_WARPS ? s_sum[lane] : 0ull;
      unsigned long long inc = x;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const int w = __ffs(__ballot_sync(0xffffffffu, before + inc > mark)) - 1;
      unsigned long long at = before + __shfl_sync(0xffffffffu, inc - x, w);
      const int s0 = (rank * VERIFY_WARPS + w) * a.seg, s1 = min(a.V, s0 + a.seg);
      for (int v = s0; v < s1; v += 32 * VEC) {
        unsigned long long y[VEC], c = 0;
        weights(v + lane * VEC, y);
#pragma unroll
        for (int e = 0; e < VEC; ++e) c += y[e];
        unsigned long long end = c;
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long z = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end += z;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, at + end > mark);
        if (hit) {
          const int l = __ffs(hit) - 1;
          unsigned long long z = at + end - c;
          int e = 0;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            z += y[i];
            e += z <= mark;
          }
          tok = v + l * VEC + __shfl_sync(0xffffffffu, e, l);
          break;
        }
        at += __shfl_sync(0xffffffffu, end, 31);
      }
    }
    for (int i = lane; i <= a.G; i += 32)
      a.tokens[(int64_t)b * (a.G + 1) + i] = i < acc ? a.drafts[(int64_t)b * a.G + i] : (i == acc ? tok : -1);
    if (lane == 0) a.accepted[b] = acc;
  }
  cluster_wait();  // no CTA leaves while another may read its total
}

}  // namespace ta
