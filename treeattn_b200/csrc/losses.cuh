// The clipped policy loss with its KL term over a vocabulary's logits, and the tokens' log-probabilities; with gradients.
//   logp = z_y / tau - log sum_j exp(z_j / tau),  rho = exp(logp - old)
//   term = -min(rho A, clip(rho, lo, hi) A) + kl (exp(ref - logp) - (ref - logp) - 1),  loss = sum over rows of w term
//   slope = dloss / dlogp = w (-A rho [not clipped] + kl (1 - exp(ref - logp))),  dloss / dz_j = slope / tau ([j = y] - p_j)
// Everything about a row but its softmax is a handful of scalars, so the gradient's factor is known as soon as the row's sum is: a
// row is read once, stays in shared memory, and its gradient is written from there. The floor is one read and one write of the
// logits; a gradient that waits for the backward pass (16-bit floats of 5 exponent bits, which need the loss's scale
// before they are rounded) reads them twice.
#pragma once
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

constexpr float LOG2E = 1.4426950408889634f;

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

// exp2((z - top) k) of a piece's elements, two at a time (packed arithmetic). The difference comes first: z k - top k, one operation, is off by
// a step of top k in every element alike, and overflows where k tops the range.
template <int N>
__device__ __forceinline__ void exp_piece(float (&z)[N], float top, float k) {
  uint64_t t2, k2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(t2) : "f"(-top));
  asm("mov.b64 %0, {%1, %1};" : "=l"(k2) : "f"(k));
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    uint64_t x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(z[i]), "f"(z[i + 1]));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(t2));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(k2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(z[i]), "=f"(z[i + 1]) : "l"(x));
    z[i] = exp2_fast(z[i]);
    z[i + 1] = exp2_fast(z[i + 1]);
  }
}

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// A row in 16-byte pieces from the boundary before its first element on: piece j holds elements [j N - lead, (j + 1) N - lead).
// Pieces that reach beyond the row are read and written element by element.
template <typename T>
struct RowPieces {
  static constexpr int N = Piece<T>::N;
  const T* row;
  int lead, V, pieces;
  __device__ __forceinline__ RowPieces(const T* r, int v) : row(r), V(v) {
    lead = (int)((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    pieces = (V + lead + N - 1) / N;
  }
  __device__ __forceinline__ bool whole(int j) const { return j * N >= lead && (j + 1) * N - lead <= V; }
  __device__ __forceinline__ uint4 edge(int j) const {  // -inf beyond the row
    uint4 v = make_uint4(Piece<T>::lowest(), Piece<T>::lowest(), Piece<T>::lowest(), Piece<T>::lowest());
    T* e = reinterpret_cast<T*>(&v);
    for (int i = 0; i < N; ++i) {
      const int at = j * N - lead + i;
      if (at >= 0 && at < V) e[i] = row[at];
    }
    return v;
  }
  __device__ __forceinline__ uint4 load(int j) const {
    return whole(j) ? load_once(reinterpret_cast<const uint4*>(row - lead) + j) : edge(j);
  }
};

template <int THREADS, typename F>
__device__ __forceinline__ float block_reduce(float x, float* shared, F op) {
  constexpr int WARPS = THREADS / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = shared[threadIdx.x & (WARPS - 1)];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// A row's gradient: f times exp2((z - top) k) taken off, `slope` added at element y. Where the output's row lies against 16-byte
// boundaries as the input's does it is written in pieces, otherwise element by element.
template <typename T>
struct GradRow {
  static constexpr int N = Piece<T>::N;
  const RowPieces<T>& r;
  T* out;
  bool same;
  float k, top, f, slope;
  int yj;
  __device__ __forceinline__ GradRow(const RowPieces<T>& r_, T* o, float top_, float k_, float f_, float s, int y)
      : r(r_), out(o), k(k_), top(top_), f(f_), slope(s), yj(y + r_.lead) {
    same = (((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(r.row)) & 15u) == 0);
  }
  __device__ __forceinline__ void put(int j, const uint4& piece) const {
    float z[N];
    Piece<T>::widen(piece, z);
    exp_piece(z, top, k);
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] *= -f;
    if (yj >= j * N && yj < (j + 1) * N) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (yj - j * N == i) z[i] += slope;
    }
    store(j, Piece<T>::narrow(z));
  }
  __device__ __forceinline__ void store(int j, const uint4& v) const {
    if (same && r.whole(j)) {
      reinterpret_cast<uint4*>(out - r.lead)[j] = v;
    } else {
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = j * N - r.lead + i;
        if (at >= 0 && at < r.V) out[at] = e[i];
      }
    }
  }
};

template <typename T, int THREADS>
__device__ __forceinline__ void write_zeros(const RowPieces<T>& r, T* out, int j0, int j1) {
  const GradRow<T> g(r, out, 0.f, 0.f, 0.f, 0.f, -1);
  for (int j = j0 + threadIdx.x; j < j1; j += THREADS) g.store(j, make_uint4(0u, 0u, 0u, 0u));
}

// A cluster of CTAs takes a row, each a share of its pieces in shared memory: read and compared, summed about the share's own
// maximum, the shares' (maximum, sum) met through distributed shared memory, the gradient written. exp is evaluated twice an element, to
// keep 16 bits of it in shared memory instead of 32 and two CTAs on an SM: one reads its row while the other computes.
template <typename T, int THREADS, bool POLICY>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) loss_kernel(const __grid_constant__ LossParams a) {
  extern __shared__ uint4 s_row[];
  __shared__ float s_red[2][THREADS / 32];
  __shared__ float s_share[2];  // this CTA's maximum and sum
  __shared__ float s_row_of[3];  // factor of the CTA's exponentials, slope / tau
  const int cs = cluster_nctarank(), rank = cluster_ctarank();
  const int64_t r = blockIdx.x / cs;
  const int b = (int)(r / a.T), t = (int)(r - (int64_t)b * a.T);
  const T* row = reinterpret_cast<const T*>(a.z) + b * a.z_sb + t * a.z_st;
  T* out = reinterpret_cast<T*>(a.grad) + b * a.g_sb + t * a.g_st;
  const RowPieces<T> p(row, a.V);
  const int j0 = min(rank * a.per, p.pieces), j1 = min(j0 + a.per, p.pieces);
  const float k = a.inv_tau * LOG2E;
  pdl_wait();
  pdl_launch_dependents();
  float w = 1.f;
  if (POLICY) {
    w = a.weight.p ? a.weight.at(b, t) : a.w0;
    if (w == 0.f) {  // not counted, whatever is in it (the same in all threads of the cluster)
      if (a.grad) write_zeros<T, THREADS>(p, out, j0, j1);
      if (rank == 0 && threadIdx.x == 0) a.logp[r] = a.top[r] = a.tot[r] = a.slope[r] = a.term[r] = 0.f;
      return;
    }
  }
  // the row's scalars, while it is read
  int64_t y = -1;
  float zy = 0.f, old = 0.f, adv = 0.f, ref = 0.f;
  if (threadIdx.x == 0) {
    y = a.tokens[b * a.t_sb + t * a.t_st];
    if (POLICY) {
      old = a.old.at(b, t);
      adv = a.adv.at(b, t);
      if (a.kl != 0.f) ref = a.ref.at(b, t);
    }
    if (y < 0 || y >= a.V) {
      if (rank == 0) record_error(DEV_INDEX_RANGE, K_LOSS, (int)r, (int)y);
      y = -1;
      zy = __int_as_float(0x7fc00000);
    } else {
      zy = to_f32(row[y]);
    }
  }
  uint32_t top = Piece<T>::lowest();
  {
    constexpr int U = 4;
    int j = j0 + threadIdx.x;
    for (; j + (U - 1) * THREADS < j1; j += U * THREADS) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = p.load(j + u * THREADS);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s_row[j - j0 + u * THREADS] = v[u];
        top = Piece<T>::max2(top, Piece<T>::max2(Piece<T>::max2(v[u].x, v[u].y), Piece<T>::max2(v[u].z, v[u].w)));
      }
    }
    for (; j < j1; j += THREADS) {
      const uint4 v = p.load(j);
      s_row[j - j0] = v;
      top = Piece<T>::max2(top, Piece<T>::max2(Piece<T>::max2(v.x, v.y), Piece<T>::max2(v.z, v.w)));
    }
  }
  auto larger = [](float x, float z) { return fmaxf(x, z); };
  auto plus = [](float x, float z) { return x + z; };
  float m = block_reduce<THREADS>(Piece<T>::top(top), s_red[0], larger);
  if (m == -INFINITY) m = 0.f;  // nothing to take off: every exponential is 0
  float sum = 0.f;
  for (int j = j0 + threadIdx.x; j < j1; j += THREADS) {
    float z[Piece<T>::N];
    Piece<T>::widen(s_row[j - j0], z);
    exp_piece(z, m, k);
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) part += z[i];
    sum += part;
  }
  sum = block_reduce<THREADS>(sum, s_red[1], plus);
  if (cs > 1) {
    if (threadIdx.x == 0) {
      s_share[0] = m;
      s_share[1] = sum;
    }
    cluster_sync_all();
  }
  if (threadIdx.x == 0) {
    float gm = m, gs = sum;
    if (cs > 1) {
      gm = -INFINITY;
      for (int c = 0; c < cs; ++c)
        if (cluster_map(s_share, c)[1] != 0.f) gm = fmaxf(gm, cluster_map(s_share, c)[0]);  // (an empty share's 0 does not count)
      if (gm == -INFINITY) gm = 0.f;
      gs = 0.f;
      for (int c = 0; c < cs; ++c) {
        const float sc = cluster_map(s_share, c)[1];
        if (sc != 0.f) gs += sc * exp2f((cluster_map(s_share, c)[0] - gm) * k);
      }
    }
    const float logp = (zy - gm) * a.inv_tau - logf(gs);
    float slope = 0.f;
    if (POLICY) {
      const float rho = expf(logp - old);
      const float held = rho < a.lo ? a.lo : rho > a.hi ? a.hi : rho;  // (comparisons that keep a NaN)
      const float free_ = rho * adv, kept = held * adv;
      float term = -(kept < free_ ? kept : free_);
      slope = (adv > 0.f ? rho > a.hi : rho < a.lo) ? 0.f : -adv * rho;
      if (a.kl != 0.f) {
        const float d = ref - logp, e = expm1f(d);
        term += a.kl * (e - d);
        slope -= a.kl * e;
      }
      slope *= w * a.inv_tau;
      if (rank == 0) {
        a.slope[r] = slope;
        a.term[r] = w * term;
      }
    }
    if (rank == 0) {
      a.logp[r] = logp;
      a.top[r] = gm;
      a.tot[r] = gs;
    }
    s_row_of[0] = sum == 0.f && gs > 0.f ? 0.f : slope * exp2f((m - gm) * k) / gs;
    s_row_of[1] = slope;
    s_row_of[2] = __int_as_float((int)y);
  }
  __syncwarp();
  if (cs > 1) cluster_arrive();  // this CTA has read the others' shares
  if (POLICY && a.grad) {
    __syncthreads();
    const float f = s_row_of[0], slope = s_row_of[1];
    if (slope == 0.f) {
      write_zeros<T, THREADS>(p, out, j0, j1);
    } else {
      const GradRow<T> g(p, out, m, k, f, slope, __float_as_int(s_row_of[2]));
      for (int j = j0 + threadIdx.x; j < j1; j += THREADS) g.put(j, s_row[j - j0]);
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
  int chunks;  // CTAs of a row
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
  const int64_t items = (int64_t)a.B * a.T * a.chunks;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int64_t r = i / a.chunks;
    const int b = (int)(r / a.T), t = (int)(r - (int64_t)b * a.T);
    const RowPieces<T> p(reinterpret_cast<const T*>(a.z) + b * a.z_sb + t * a.z_st, a.V);
    T* out = reinterpret_cast<T*>(a.grad) + b * a.g_sb + t * a.g_st;
    const int j0 = (int)(i - r * a.chunks) * GRAD_PIECES, j1 = min(j0 + GRAD_PIECES, p.pieces);
    const float own = a.slope.at(b, t);
    const float slope = own == 0.f ? 0.f : own * a.by * up;
    if (own == 0.f) {
      write_zeros<T, GRAD_THREADS>(p, out, j0, j1);
      continue;
    }
    const int64_t y = a.tokens[b * a.t_sb + t * a.t_st];
    const float f = y >= 0 && y < a.V ? slope / a.tot[r] : __int_as_float(0x7fc00000);
    const GradRow<T> g(p, out, a.top[r], a.inv_tau * LOG2E, f, slope, (int)y);
    uint4 v[GRAD_PIECES / GRAD_THREADS];
#pragma unroll
    for (int u = 0; u < GRAD_PIECES / GRAD_THREADS; ++u) {
      const int j = j0 + threadIdx.x + u * GRAD_THREADS;
      if (j < j1) v[u] = p.load(j);
    }
#pragma unroll
    for (int u = 0; u < GRAD_PIECES / GRAD_THREADS; ++u) {
      const int j = j0 + threadIdx.x + u * GRAD_THREADS;
      if (j < j1) g.put(j, v[u]);
    }
  }
}

}  // namespace ta
