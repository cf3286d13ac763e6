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

constexpr int VERIFY_THREADS = 1024;

struct VerifyParams {
  const void *p, *q;
  int64_t p_sb, p_sr, q_sb, q_sr;
  const int64_t* drafts;  // (B, G)
  const float* u;         // (B, G + 1): one for each draft, the last for the draw
  const int32_t* n;       // (B,) drafts of each sequence, or null (G)
  int B, G, V;
  int64_t* tokens;        // (B, G + 1)
  int32_t* accepted;      // (B,)
};

// max(p - q, 0) in steps of 2^-38; what is not a number weighs nothing
__device__ __forceinline__ unsigned long long left_over(float p, float q) {
  const float d = p > q ? fminf(__fsub_rn(p, q), 1.f) : 0.f;
  return (unsigned long long)(d * 274877906944.f);
}

template <typename T>
__global__ void __launch_bounds__(VERIFY_THREADS) verify_kernel(VerifyParams a) {
  __shared__ int s_acc;
  __shared__ unsigned long long s_sum[2][32];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* P = reinterpret_cast<const T*>(a.p) + b * a.p_sb;
  const T* Q = reinterpret_cast<const T*>(a.q) + b * a.q_sb;
  if (tid == 0) s_acc = 0x7fffffff;
  __syncthreads();
  int n = a.n ? a.n[b] : a.G;
  if (n < 0 || n > a.G) {
    if (tid == 0) record_error(DEV_INDEX_RANGE, K_VERIFY, b, n);
    n = n < 0 ? 0 : a.G;
  }
  for (int i = tid; i < n; i += VERIFY_THREADS) {
    const int64_t d = a.drafts[(int64_t)b * a.G + i];
    bool ok = false;
    if (d < 0 || d >= a.V)
      record_error(DEV_INDEX_RANGE, K_VERIFY, b, (int)d);
    else
      ok = __fmul_rn(a.u[(int64_t)b * (a.G + 1) + i], to_f32(Q[i * a.q_sr + d])) < to_f32(P[i * a.p_sr + d]);
    if (!ok) atomicMin(&s_acc, i);
  }
  __syncthreads();
  const int acc = min(s_acc, n);
  const T* pr = P + acc * a.p_sr;
  const T* qr = acc < n ? Q + acc * a.q_sr : nullptr;
  // warp w owns the words [w seg, (w + 1) seg)
  const int seg = ((a.V + 31) / 32 + 31) / 32 * 32;
  const int v0 = warp * seg, v1 = min(a.V, v0 + seg);
  unsigned long long left = 0, whole = 0;
  for (int v = v0 + lane; v < v1; v += 32) {
    const float x = to_f32(pr[v]);
    whole += left_over(x, 0.f);
    if (qr) left += left_over(x, to_f32(qr[v]));
  }
  for (int o = 16; o > 0; o >>= 1) {
    left += __shfl_xor_sync(0xffffffffu, left, o);
    whole += __shfl_xor_sync(0xffffffffu, whole, o);
  }
  if (lane == 0) {
    s_sum[0][warp] = left;
    s_sum[1][warp] = whole;
  }
  __syncthreads();
  if (warp == 0) {
    unsigned long long x = s_sum[0][lane];
    unsigned long long tl = x;
    for (int o = 16; o > 0; o >>= 1) tl += __shfl_xor_sync(0xffffffffu, tl, o);
    const bool rest = tl > 0;
    if (!rest) x = s_sum[1][lane];
    unsigned long long inc = x;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const unsigned long long tot = __shfl_sync(0xffffffffu, inc, 31);
    const float uf = a.u[(int64_t)b * (a.G + 1) + a.G];
    const unsigned long long u24 = uf > 0.f ? (unsigned long long)min(uf * 16777216.f, 16777215.f) : 0ull;
    const unsigned long long mark = (tot >> 24) * u24 + (((tot & 0xffffffull) * u24) >> 24);
    const uint32_t past = __ballot_sync(0xffffffffu, inc > mark);
    int64_t tok = a.V - 1;
    if (past) {
      const int w = __ffs(past) - 1;
      unsigned long long at = __shfl_sync(0xffffffffu, inc - x, w);
      const int e = min(a.V, (w + 1) * seg);
      for (int v = w * seg; v < e; v += 32) {
        unsigned long long y = 0;
        if (v + lane < e) y = left_over(to_f32(pr[v + lane]), rest ? to_f32(qr[v + lane]) : 0.f);
        unsigned long long c = y;
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long z = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) c += z;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, at + c > mark);
        if (hit) {
          tok = v + __ffs(hit) - 1;
          break;
        }
        at += __shfl_sync(0xffffffffu, c, 31);
      }
    }
    for (int i = lane; i <= a.G; i += 32)
      a.tokens[(int64_t)b * (a.G + 1) + i] = i < acc ? a.drafts[(int64_t)b * a.G + i] : (i == acc ? tok : -1);
    if (lane == 0) a.accepted[b] = acc;
  }
}

}  // namespace ta
