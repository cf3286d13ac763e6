// The clipped policy loss with its KL term over a vocabulary's logits, and the tokens' log-probabilities; with gradients.
//   logp = z_y / tau - log sum_j exp(z_j / tau),  rho = exp(logp - old)
//   term = -min(rho A, clip(rho, lo, hi) A) + kl (exp(ref - logp) - (ref - logp) - 1),  loss = sum over rows of w term
//   slope = dloss / dlogp = w (-A rho [not clipped] + kl (1 - exp(ref - logp))),  dloss / dz_j = slope / tau ([j = y] - p_j)
// Everything about a row but its softmax is a handful of scalars, so the gradient's factor is known as soon as the row's sum is: a
// row is read once, stays in shared memory, and the gradient is written from there. The floor is one read and one write of the
// logits; a gradient that waits for the backward pass (16-bit floats of 5 exponent bits, which need the loss's scale
// before they are rounded) reads them twice.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace ta {

// A vector of floats by (b, t), any strides; null where there is none.
struct RowVec {
  const float* p;
  int64_t sb, st;
  __device__ __forceinline__ float at(int b, int t) const { return p[b * sb + t * st]; }
};

struct LossParams {
  const void* z;
  int64_t z_sb, z_st;
  int B, T, V;
  int per;  // 16-byte pieces of a CTA's share of a row
  const int64_t* tokens;
  int64_t t_sb, t_st;
  RowVec old, adv, ref, weight;
  float w0, lo, hi, kl, inv_tau;
  float *logp, *top, *tot, *slope, *term;  // (rows,): the last three, of which slope and term belong to the policy loss
  void* grad;                              // null: none now
  int64_t g_sb, g_st;
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// The two elements of a word of a 16-byte piece, as fp32; a piece of fp32 has one a word.
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint32_t lowest() { return 0xff800000u; }
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 narrow(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  // running maximum of words (a NaN loses: it is found in the sum)
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t a) { return __uint_as_float(a); }
};
template <typename H, typename H2> struct Piece16 {
  static constexpr int N = 8;
  static __device__ __forceinline__ H2 as2(uint32_t a) { return *reinterpret_cast<H2*>(&a); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    H2 m = __hmax2(as2(a), as2(b));
    return *reinterpret_cast<uint32_t*>(&m);
  }
  static __device__ __forceinline__ float top(uint32_t a) { return fmaxf(to_f32(as2(a).x), to_f32(as2(a).y)); }
};
template <> struct Piece<__nv_bfloat16> : Piece16<__nv_bfloat16, __nv_bfloat162> {
  static __device__ __forceinline__ uint32_t lowest() { return 0xff80ff80u; }
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 narrow(const float (&f)[8]) {
    uint4 v;
    store_vec_from_f32<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16*>(&v), f);
    return v;
  }
};
template <> struct Piece<__half> : Piece16<__half, __half2> {
  static __device__ __forceinline__ uint32_t lowest() { return 0xfc00fc00u; }
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[8]) {
    load_vec_f32<__half>(reinterpret_cast<const __half*>(&v), f);
  }
  static __device__ __forceinline__ uint4 narrow(const float (&f)[8]) {
    uint4 v;
    store_vec_from_f32<__half>(reinterpret_cast<__half*>(&v), f);
    return v;
  }
};

__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; 0 at -inf, NaN at NaN
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A reference logit m that exponentials are taken about: exp2(z k - R), R = m k rounded: one operation and the exponential. R is the
// reference as it stands (the rounding of m k puts one factor on all of its exponentials), and whatever is compared with it takes R
// itself, so that the factor cancels. From 2^20 on, where that factor may pass 2^(1/16) and further up leave the range (a word banned by a finite
// -1e10: 2^439), the difference is taken first and the reference is m k.
struct Ref {
  float m, off;  // off = -R
  bool far;
  __device__ __forceinline__ Ref(float m_, float k) : m(m_), off(-m_ * k), far(!(fabsf(off) < 1048576.f)) {}
  __device__ __forceinline__ float of(float z, float k) const { return far ? (z - m) * k : fmaf(z, k, off); }
  // what a sum about o is multiplied by to be one about this: each as it stands, R or m k
  __device__ __forceinline__ float from(const Ref& o, float k) const {
    if (!far) return exp2_fast(o.far ? fmaf(o.m, k, off) : off - o.off);
    return exp2_fast(o.far ? (o.m - m) * k : -fmaf(m, k, o.off));
  }
};

// A piece that is read once. Volatile, with memory as a clobber, and not through the read-only path: the launch before this one may write
// the logits until pdl_wait returns, and nothing else keeps a load of an address that is known before from being moved above it.
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// The element at a time forms of a piece that reaches beyond its row (elements [0, V) of it; the piece's first is `at`): -inf there.
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* row, int at, int V) {
  uint4 v = make_uint4(Piece<T>::lowest(), Piece<T>::lowest(), Piece<T>::lowest(), Piece<T>::lowest());
  T* e = reinterpret_cast<T*>(&v);
  for (int i = 0; i < Piece<T>::N; ++i)
    if (at + i >= 0 && at + i < V) e[i] = row[at + i];
  return v;
}
template <typename T>
__device__ __noinline__ void store_edge(T* row, int at, int V, uint4 v) {
  const T* e = reinterpret_cast<const T*>(&v);
  for (int i = 0; i < Piece<T>::N; ++i)
    if (at + i >= 0 && at + i < V) row[at + i] = e[i];
}

// A row in 16-byte pieces from the boundary before its first element on: piece j holds elements [j N - lead, (j + 1) N - lead).
// Pieces that reach beyond the row are read and written element by element.
template <typename T>
struct RowPieces {
  static constexpr int N = Piece<T>::N;
  const T* row;
  int lead, V, pieces;
  int first, last;  // the pieces that reach beyond the row, or -1
  __device__ __forceinline__ RowPieces(const T* r, int v, bool aligned = false) : row(r), V(v) {
    lead = aligned ? 0 : (int)((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    pieces = (V + lead + N - 1) / N;
    first = lead ? 0 : -1;
    last = (V + lead) % N ? pieces - 1 : -1;
  }
  __device__ __forceinline__ bool whole(int j) const { return j != first && j != last; }
  __device__ __forceinline__ uint4 edge(int j) const { return load_edge(row, j * N - lead, V); }
  __device__ __forceinline__ const uint4* at(int j) const { return reinterpret_cast<const uint4*>(row - lead) + j; }
  __device__ __forceinline__ uint4 load(int j) const { return whole(j) ? load_once(at(j)) : edge(j); }
};

// A row's gradient. Where it lies against 16-byte boundaries as the row itself does it is written in pieces, otherwise element by
// element.
template <typename T, bool ALIGNED>
struct GradRow {
  static constexpr int N = Piece<T>::N;
  const RowPieces<T>& r;
  T* out;
  bool same;
  __device__ __forceinline__ GradRow(const RowPieces<T>& r_, T* o) : r(r_), out(o) {
    same = (((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(r.row)) & 15u) == 0);
  }
  __device__ __forceinline__ void edge(int j, const uint4& v) const { store_edge(out, j * N - r.lead, r.V, v); }
  __device__ __forceinline__ void whole(int j, const uint4& v) const {  // a piece that lies in the row
    if (ALIGNED || same)
      reinterpret_cast<uint4*>(out - r.lead)[j] = v;
    else
      edge(j, v);
  }
  __device__ __forceinline__ void zeros(int j0, int j, int end, int step, int cut) const {
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (; j < end; j += step) whole(j0 + j, zero);
    if (cut >= 0) edge(j0 + cut, zero);
  }
};

// A softmax's sum about a reference: s = sum of exp2(z k - m k). Empty (s = 0) it has no reference.
struct Share {
  float m, s;
};

// The warp's shares as one, in every lane and one order.
__device__ __forceinline__ Share warp_share(const Share& x, float k) {
  float m = x.s == 0.f ? -INFINITY : x.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m == -INFINITY) m = 0.f;
  float s = x.s == 0.f ? 0.f : x.s * Ref(m, k).from(Ref(x.m, k), k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return {m, s};
}

// A cluster of CTAs takes a row, each a share of its pieces. All of a share is asked for at once and lies in shared memory; a thread
// copies the pieces that it will look at itself, so that no barrier is needed for them. It sums exponentials about the largest element
// of its first piece; where that was a poor choice (the sum leaves [1/2, 2^100]) it looks for its largest element and sums again. The
// warps' and CTAs' (reference, sum) meet in one step, one thread works out the row's scalars, and the gradient is written from the share:
// exp2(z k - m k + log2(slope / sum)) in 16 bits, one operation, the exponential and the rounding an element, and slope / sum exp2(z k - m k) in
// 32, where the sum's rounding would be seen (2048 x 50304 fp32: 156 us; 168 with the factor in the exponent). exp is evaluated twice, to keep
// 16 bits of an element instead of 32 and two CTAs on an SM: one waits for its row while the other computes. (Kept in registers
// instead, with the next row read ahead, an element costs less, but the CTAs that a row then needs wait for each other: 810 us against 290
// for 8 x 1024 x 50304 bf16, a quarter of it not counted.)
// Without a gradient nothing is kept, and the row is summed as it arrives: 8192 rows of 50304 bf16 in 133 us, 6.2 TB/s. With it 2048 rows
// take 86 us (with the loss's sum behind them), 4.8 TB/s read and written, the issue slots half full: it is the two CTAs' phases that do not
// always overlap.
// ALIGNED: every row begins and ends on a 16-byte boundary, in the gradient too.
// (Six CTAs of 256 threads on an SM where that costs nothing else, five otherwise: 8192 x 50304 bf16 133 against 135 us, 2048 x 50304 fp32 76
// against 74.)
template <typename T, int THREADS, int MODE, bool ALIGNED>  // MODE 0: log-probabilities, 1: the policy loss, 2: and its gradient
__global__ void __launch_bounds__(THREADS, (MODE == 2 ? 1024 : MODE == 0 && ALIGNED && sizeof(T) == 2 ? 1536 : 1280) / THREADS)
    loss_kernel(const __grid_constant__ LossParams a) {
  constexpr int N = Piece<T>::N, WARPS = THREADS / 32, U = 4;
  constexpr bool POLICY = MODE > 0, KEEP = MODE == 2;
  extern __shared__ uint4 share[];
  __shared__ Share s_warp[WARPS];
  __shared__ float s_of[4];  // of the row: reference, factor of the exponentials, its logarithm (base 2) and slope / tau
  __shared__ int s_token;
  const int tid = threadIdx.x, cs = cluster_nctarank(), rank = cluster_ctarank();
  const int r = blockIdx.x / cs;
  const int b = r / a.T, t = r - b * a.T;
  const T* const row = reinterpret_cast<const T*>(a.z) + b * a.z_sb + t * a.z_st;
  const float k = a.inv_tau * LOG2E;
  const RowPieces<T> p(row, a.V, ALIGNED);
  const int j0 = rank * a.per, n = min(a.per, p.pieces - j0);  // (n < 1: a share without pieces)
  // the share's whole pieces are [i0, i1); one that the row begins or ends in belongs to a thread of the second or third warp (the first has
  // the row's scalars to read)
  const int i0 = !ALIGNED && n > 0 && p.first == j0, i1 = !ALIGNED && p.last == j0 + n - 1 && n > i0 ? n - 1 : n;
  const int edge = ALIGNED ? -1 : tid == 32 && i0 ? 0 : tid == 64 && n > 0 && i1 < n ? n - 1 : -1;
  pdl_wait();
  pdl_launch_dependents();
  T* const out = MODE == 2 ? reinterpret_cast<T*>(a.grad) + b * a.g_sb + t * a.g_st : nullptr;
  const GradRow<T, ALIGNED> g(p, out);
  float w = 1.f;
  if (POLICY) {
    w = a.weight.p ? a.weight.at(b, t) : a.w0;
    if (w == 0.f) {  // not counted, whatever is in it (the same in all threads of the cluster)
      if (MODE == 2) g.zeros(j0, i0 + tid, i1, THREADS, edge);
      if (rank == 0 && tid == 0) a.logp[r] = a.top[r] = a.tot[r] = a.slope[r] = a.term[r] = 0.f;
      return;
    }
  }
  const uint4* const from = p.at(j0);
  if (KEEP) {
    for (int j = i0 + tid; j < i1; j += THREADS)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(share + j)), "l"(from + j) : "memory");
    if (edge >= 0) share[edge] = p.edge(j0 + edge);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the row's scalars, while it arrives
  int64_t y = -1;
  T zy = from_f32<T>(0.f);
  float old = 0.f, adv = 0.f, ref = 0.f;
  if (tid == 0) y = a.tokens[b * a.t_sb + t * a.t_st];
  auto scalars = [&]() {
    if (tid != 0) return;
    if (POLICY) {
      old = a.old.at(b, t);
      adv = a.adv.at(b, t);
      if (a.kl != 0.f) ref = a.ref.at(b, t);
    }
    if (y < 0 || y >= a.V) {
      if (rank == 0) record_error(DEV_INDEX_RANGE, K_LOSS, r, (int)y);
      y = -1;
    } else {
      zy = row[y];
    }
  };
  if (KEEP) {
    scalars();
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  auto piece = [&](int j) { return KEEP ? share[j] : load_once(from + j); };  // a whole one
  auto largest = [](const uint4& v) { return Piece<T>::top(Piece<T>::max2(Piece<T>::max2(v.x, v.y), Piece<T>::max2(v.z, v.w))); };
  auto piece_sum = [&](const uint4& v, const Ref& m) {
    float z[N];
    Piece<T>::widen(v, z);
    if (!m.far) {
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = exp2_fast(fmaf(z[i], k, m.off));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = exp2_fast((z[i] - m.m) * k);
    }
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; ++i) z[i] += z[i + o];
    return z[0];
  };
  auto sum_about = [&](const Ref& m, int j, float s) {
    if (!KEEP) {
      for (; j + (U - 1) * THREADS < i1; j += U * THREADS) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = piece(j + u * THREADS);
#pragma unroll
        for (int u = 0; u < U; ++u) s += piece_sum(v[u], m);
      }
    }
    for (; j < i1; j += THREADS) s += piece_sum(piece(j), m);
    return s;
  };
  float top = 0.f, s = 0.f;
  const int first = i0 + tid;
  uint4 v[U], cut;
  if (!KEEP) {  // the first pieces are asked for before anything is waited for, the scalars then
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * THREADS < i1) v[u] = piece(first + u * THREADS);
    scalars();
  }
  if (edge >= 0) cut = KEEP ? share[edge] : p.edge(j0 + edge);
  if (first < i1 || edge >= 0) {
    top = largest(first < i1 ? KEEP ? piece(first) : v[0] : cut);
    if (!(top > -INFINITY)) top = 0.f;  // nothing to take off
    const Ref m(top, k);
    if (!KEEP) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + u * THREADS < i1) s += piece_sum(v[u], m);
    }
    s = sum_about(m, KEEP ? first : first + U * THREADS, s);
    if (edge >= 0) s += piece_sum(cut, m);
    if (!(s >= 0.5f && s < 1.2676506e30f)) {
      top = edge >= 0 ? largest(cut) : -INFINITY;
      for (int j = first; j < i1; j += THREADS) top = fmaxf(top, largest(piece(j)));
      if (!(top > -INFINITY)) top = 0.f;
      const Ref again(top, k);
      s = sum_about(again, first, 0.f);
      if (edge >= 0) s += piece_sum(cut, again);
    }
  }
  __syncwarp();
  const Share mine = warp_share({top, s}, k);
  if ((tid & 31) == 0) s_warp[tid >> 5] = mine;
  if (cs > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (tid < 32) {
    Share sum = {0.f, 0.f};
    for (int i = tid; i < cs * WARPS; i += 32) {
      const Share x = (cs > 1 ? cluster_map(s_warp, i / WARPS) : s_warp)[i % WARPS];
      if (x.s != 0.f) {
        if (sum.s == 0.f) {
          sum = x;
        } else if (x.m > sum.m) {
          sum.s = sum.s * Ref(x.m, k).from(Ref(sum.m, k), k) + x.s;
          sum.m = x.m;
        } else {
          sum.s += x.s * Ref(sum.m, k).from(Ref(x.m, k), k);
        }
      }
    }
    sum = warp_share(sum, k);
    if (tid == 0) {
      const float logp = Ref(sum.m, k).of(y < 0 ? __int_as_float(0x7fc00000) : to_f32(zy), k) * LN2 - logf(sum.s);
      float slope = 0.f;
      if (POLICY) {
        const float rho = expf(logp - old);
        const float held = rho < a.lo ? a.lo : rho > a.hi ? a.hi : rho;  // (comparisons that keep a NaN)
        const float free_ = rho * adv, kept = held * adv;
        float term = -(kept < free_ ? kept : free_);
        slope = (adv > 0.f ? rho > a.hi : adv <= 0.f && rho < a.lo) ? 0.f : -adv * rho;  // (NaN where A is)
        if (a.kl != 0.f) {
          const float d = ref - logp, x = expm1f(d);
          term += a.kl * (x - d);
          slope -= a.kl * x;
        }
        slope *= w * a.inv_tau;
        if (rank == 0) {
          a.slope[r] = slope;
          a.term[r] = w * term;
        }
        const float f = slope / sum.s;
        s_of[0] = sum.m;
        s_of[1] = -f;
        s_of[2] = log2f(fabsf(f));
        s_of[3] = slope;
        s_token = (int)y;
      }
      if (rank == 0) {
        a.logp[r] = logp;
        a.top[r] = sum.m;
        a.tot[r] = sum.s;
      }
    }
    __syncwarp();
  }
  if (cs > 1) cluster_arrive();  // this CTA has read the others' shares
  if (MODE == 2) {
    __syncthreads();
    const float slope = s_of[3];
    const Ref m(s_of[0], k);
    const int yt = s_token, yp = yt < 0 ? -1 : (yt + p.lead) / N - j0, yi = (yt + p.lead) % N;
    auto add = [&](int j, float (&z)[N]) {
      if (j == yp) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (yi == i) z[i] += slope;
      }
    };
    if (slope == 0.f) {
      g.zeros(j0, first, i1, THREADS, edge);
    } else if (sizeof(T) == 4 || !(fabsf(m.off) + fabsf(s_of[2]) < 256.f)) {
      // the factor after the exponential: exact to fp32's steps wherever the row lies
      const float f = s_of[1];
      auto all = [&](auto far) {
        auto one = [&](int j) {
          float z[N];
          Piece<T>::widen(share[j], z);
#pragma unroll
          for (int i = 0; i < N; ++i) z[i] = f * exp2_fast(decltype(far)::value ? (z[i] - m.m) * k : fmaf(z[i], k, m.off));
          add(j, z);
          return Piece<T>::narrow(z);
        };
        for (int j = first; j < i1; j += THREADS) g.whole(j0 + j, one(j));
        if (edge >= 0) g.edge(j0 + edge, one(edge));
      };
      if (m.far)
        all(std::true_type());
      else
        all(std::false_type());
    } else {
      // 16 bits: the factor joins the exponent. Their sum is rounded once more, by 2^-17 of its 256 at most: nothing beside the
      // output's 2^-12 or 2^-9.
      const float off = m.off + s_of[2];
      auto all = [&](auto sign) {
        auto one = [&](int j) {
          float z[N];
          Piece<T>::widen(share[j], z);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float e = exp2_fast(fmaf(z[i], k, off));
            z[i] = decltype(sign)::value ? -e : e;
          }
          add(j, z);
          return Piece<T>::narrow(z);
        };
        for (int j = first; j < i1; j += THREADS) g.whole(j0 + j, one(j));
        if (edge >= 0) g.edge(j0 + edge, one(edge));
      };
      if (slope > 0.f)
        all(std::true_type());
      else
        all(std::false_type());
    }
  }
  if (cs > 1) cluster_wait();
}

// loss = the terms' sum, in 64 bits and one order.
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* term, int64_t n, float* loss) {
  __shared__ double s[32];
  pdl_wait();
  pdl_launch_dependents();
  double x = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) x += (double)term[i];
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x < 32) {
    x = s[threadIdx.x];
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (threadIdx.x == 0) *loss = (float)x;
  }
}

struct LogitsGradParams {
  const void* z;
  int64_t z_sb, z_st;
  int B, T, V;
  int chunks;      // pieces of a row that CTAs take
  uint32_t items;  // and of all rows
  const int64_t* tokens;
  int64_t t_sb, t_st;
  const float *top, *tot;
  RowVec slope;
  float by, inv_tau;  // slope * by is the factor of the row
  const float* up;    // the gradient of the loss, or null (1)
  int unit_done;      // the output already holds the gradient for a factor of 1
  void* grad;
  int64_t g_sb, g_st;
};

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_PIECES = GRAD_THREADS * 4;

// The gradient of saved rows: one read, one write. Every CTA takes a piece of a row.
template <typename T>
__global__ void __launch_bounds__(GRAD_THREADS) logits_grad_kernel(const __grid_constant__ LogitsGradParams a) {
  pdl_wait();
  pdl_launch_dependents();
  const float up = a.up ? *a.up : 1.f;
  if (a.unit_done && up == 1.f) return;
  for (uint32_t i = blockIdx.x; i < a.items; i += gridDim.x) {
    const uint32_t r = i / (uint32_t)a.chunks;
    const int b = (int)(r / (uint32_t)a.T), t = (int)(r - (uint32_t)b * a.T);
    const RowPieces<T> p(reinterpret_cast<const T*>(a.z) + b * a.z_sb + t * a.z_st, a.V);
    T* out = reinterpret_cast<T*>(a.grad) + b * a.g_sb + t * a.g_st;
    const int j0 = (int)(i - r * (uint32_t)a.chunks) * GRAD_PIECES, j1 = min(j0 + GRAD_PIECES, p.pieces);
    const float own = a.slope.at(b, t);
    const int64_t y = a.tokens[b * a.t_sb + t * a.t_st];
    const bool known = y >= 0 && y < a.V;
    const float slope = own * a.by * up;
    const GradRow<T, false> g(p, out);
    const int yp = known ? ((int)y + p.lead) / Piece<T>::N : -1, yi = known ? ((int)y + p.lead) % Piece<T>::N : 0;
    constexpr int U = GRAD_PIECES / GRAD_THREADS, N = Piece<T>::N;
    uint4 v[U];
    if (own != 0.f) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + threadIdx.x + u * GRAD_THREADS;
        if (j < j1) v[u] = p.load(j);
      }
    }
    const float f = known ? -slope / a.tot[r] : __int_as_float(0x7fc00000), k = a.inv_tau * LOG2E;
    const Ref m(a.top[r], k);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + threadIdx.x + u * GRAD_THREADS;
      if (j >= j1) break;
      if (own == 0.f) {
        p.whole(j) ? g.whole(j, make_uint4(0u, 0u, 0u, 0u)) : g.edge(j, make_uint4(0u, 0u, 0u, 0u));
        continue;
      }
      float z[N];
      Piece<T>::widen(v[u], z);
      if (!m.far) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = exp2_fast(fmaf(z[i], k, m.off)) * f;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = exp2_fast((z[i] - m.m) * k) * f;
      }
      if (j == yp) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (yi == i) z[i] += slope;
      }
      if (p.whole(j))
        g.whole(j, Piece<T>::narrow(z));
      else
        g.edge(j, Piece<T>::narrow(z));
    }
  }
}

}  // namespace ta
