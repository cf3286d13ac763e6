// C ABI of the training losses over a vocabulary's logits.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "../../include/treeattn_b200.h"
#include "host.cuh"
#include "losses.cuh"

namespace ta_host {
// This translation unit's device error record (see ta_device_error), read and cleared.
cudaError_t losses_device_error(int* out4) {
  cudaError_t e = cudaMemcpyFromSymbol(out4, ta::g_dev_err, 4 * sizeof(int));
  if (e != cudaSuccess || out4[0] == 0) return e;
  const int zero[4] = {0, 0, 0, 0};
  return cudaMemcpyToSymbol(ta::g_dev_err, zero, 4 * sizeof(int));
}
}  // namespace ta_host

namespace {

using namespace ta_host;

constexpr int MAX_ROW = 1 << 20;          // bytes: a cluster of 8 holds a row
constexpr int TWO_PER_SM = 108 * 1024;    // bytes of a row in a CTA's shared memory, with two CTAs on an SM

int check_rows(const char* who, const void* z, int dtype, int B, int T, int V, const int64_t* tokens, float tau) {
  if (!valid_dtype(dtype)) return fail(TA_ERR_ARG, "%s: bad dtype %d", who, dtype);
  if (B < 0 || T < 0 || V < 1 || V > MAX_ROW / esize_of(dtype) || (int64_t)B * T > (1 << 27))
    return fail(TA_ERR_ARG, "%s: bad sizes B=%d T=%d V=%d (rows of at most %d bytes, 2^27 of them)", who, B, T, V, MAX_ROW);
  if (!(tau > 0.f) || !std::isfinite(tau) || !std::isfinite(2.f / tau))
    return fail(TA_ERR_ARG, "%s: temperature %g (positive and finite)", who, tau);
  if ((int64_t)B * T > 0 && (!z || !tokens)) return fail(TA_ERR_ARG, "%s: null pointer", who);
  return TA_OK;
}

template <typename T, int THREADS, int MODE, bool ALIGNED>
int launch_loss(const ta::LossParams& a, int cs, cudaStream_t st, const char* who) {
  static SmemAttr attr;
  const size_t smem = MODE == 2 ? (size_t)a.per * 16 : 0;
  if (int r = allow_smem(attr, ta::loss_kernel<T, THREADS, MODE, ALIGNED>, smem, who)) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.T * cs));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ta::loss_kernel<T, THREADS, MODE, ALIGNED>, a);
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  return TA_OK;
}

template <typename T, int MODE>
int run_loss(ta::LossParams& a, cudaStream_t st, const char* who) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t rows = (int64_t)a.B * a.T;
  const int pieces = (a.V + 2 * N - 2) / N;  // at most, wherever the row begins
  // CTAs of a row: as few as leave room for two on an SM (one, where nothing is kept), more where the rows do not fill the GPU
  int cs = 1;
  while (cs < 8 && ((MODE == 2 && (int64_t)pieces * 16 > (int64_t)cs * TWO_PER_SM) || (rows * cs < 2 * sm_count() && pieces * 16 >= 2 * cs * 8192)))
    cs *= 2;
  a.per = (pieces + cs - 1) / cs;
  const bool aligned = a.V % N == 0 && rows_aligned(a.z, sizeof(T), {a.z_sb, a.z_st}) &&
                       (MODE < 2 || rows_aligned(a.grad, sizeof(T), {a.g_sb, a.g_st}));
  // Small shares: 128 threads, so that more rows are under way on an SM. 8192 x 8192 bf16 with its gradient 61 us, 114 with 512 threads, without
  // it 37, 39 with 256; 16384 x 1000 fp32 56 and 165, 39 and 53; 8192 x 11000 f16 without 49 and 51. Few rows lose: 300 x 8192 bf16 without
  // 10.2 and 8.2.
  if (a.per * 16 < 24 * 1024) {
    if (aligned) return launch_loss<T, 128, MODE, true>(a, cs, st, who);
    return launch_loss<T, 128, MODE, false>(a, cs, st, who);
  }
  constexpr int WIDE = MODE == 2 ? 512 : 256;
  if (aligned) return launch_loss<T, WIDE, MODE, true>(a, cs, st, who);
  return launch_loss<T, WIDE, MODE, false>(a, cs, st, who);
}

template <int MODE>
int by_type(ta::LossParams& a, int dtype, cudaStream_t st, const char* who) {
  switch (dtype) {
    case TA_F32: return run_loss<float, MODE>(a, st, who);
    case TA_BF16: return run_loss<__nv_bfloat16, MODE>(a, st, who);
    default: return run_loss<__half, MODE>(a, st, who);
  }
}

}  // namespace

extern "C" {

int ta_token_logp(const void* logits, int dtype, int64_t z_sb, int64_t z_st, int B, int T, int V, const int64_t* tokens,
                  int64_t t_sb, int64_t t_st, float temperature, float* logp, float* stats, void* stream) {
  g_err.clear();
  const char* who = "ta_token_logp";
  if (int r = check_rows(who, logits, dtype, B, T, V, tokens, temperature)) return r;
  const int64_t rows = (int64_t)B * T;
  if (rows == 0) return TA_OK;
  if (!logp || !stats) return fail(TA_ERR_ARG, "%s: null pointer", who);
  ta::LossParams a{};
  a.z = logits; a.z_sb = z_sb; a.z_st = z_st;
  a.B = B; a.T = T; a.V = V;
  a.tokens = tokens; a.t_sb = t_sb; a.t_st = t_st;
  a.inv_tau = 1.f / temperature;
  a.logp = logp; a.top = stats; a.tot = stats + rows;
  return by_type<0>(a, dtype, S(stream), who);
}

int ta_policy_loss(const void* logits, int dtype, int64_t z_sb, int64_t z_st, int B, int T, int V, const int64_t* tokens,
                   int64_t t_sb, int64_t t_st, const float* const* by_row, const int64_t* by_row_strides, float weight0,
                   float lo, float hi, float kl, float temperature, float* loss, float* logp, float* stats, void* grad,
                   int64_t g_sb, int64_t g_st, void* stream) {
  g_err.clear();
  const char* who = "ta_policy_loss";
  if (int r = check_rows(who, logits, dtype, B, T, V, tokens, temperature)) return r;
  if (!(lo <= 1.f) || !(hi >= 1.f) || !std::isfinite(kl))
    return fail(TA_ERR_ARG, "%s: ratios clipped to [%g, %g], KL weight %g", who, lo, hi, kl);
  if (!loss) return fail(TA_ERR_ARG, "%s: null pointer", who);
  const int64_t rows = (int64_t)B * T;
  const cudaStream_t st = S(stream);
  if (rows > 0) {
    if (!by_row || !by_row_strides || !logp || !stats || !by_row[0] || !by_row[1] || (kl != 0.f && !by_row[2]))
      return fail(TA_ERR_ARG, "%s: null pointer", who);
    ta::LossParams a{};
    a.z = logits; a.z_sb = z_sb; a.z_st = z_st;
    a.B = B; a.T = T; a.V = V;
    a.tokens = tokens; a.t_sb = t_sb; a.t_st = t_st;
    ta::RowVec* const v[4] = {&a.old, &a.adv, &a.ref, &a.weight};
    for (int i = 0; i < 4; ++i) *v[i] = {by_row[i], by_row_strides[2 * i], by_row_strides[2 * i + 1]};
    a.w0 = weight0; a.lo = lo; a.hi = hi; a.kl = kl; a.inv_tau = 1.f / temperature;
    a.logp = logp; a.top = stats; a.tot = stats + rows; a.slope = stats + 2 * rows; a.term = stats + 3 * rows;
    a.grad = grad; a.g_sb = g_sb; a.g_st = g_st;
    if (int r = grad ? by_type<2>(a, dtype, st, who) : by_type<1>(a, dtype, st, who)) return r;
  }
  const cudaError_t e = launch_pdl(ta::loss_sum_kernel, dim3(1), dim3(1024), 0, st, (const float*)stats + 3 * rows, rows, loss);
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  return TA_OK;
}

int ta_logits_grad(const void* logits, int dtype, int64_t z_sb, int64_t z_st, int B, int T, int V, const int64_t* tokens,
                   int64_t t_sb, int64_t t_st, const float* stats, const float* slope, int64_t s_sb, int64_t s_st,
                   float slope_by, float temperature, const float* up, int unit_done, void* grad, int64_t g_sb,
                   int64_t g_st, void* stream) {
  g_err.clear();
  const char* who = "ta_logits_grad";
  if (int r = check_rows(who, logits, dtype, B, T, V, tokens, temperature)) return r;
  const int64_t rows = (int64_t)B * T;
  if (rows == 0) return TA_OK;
  if (!stats || !slope || !grad) return fail(TA_ERR_ARG, "%s: null pointer", who);
  ta::LogitsGradParams a{};
  a.z = logits; a.z_sb = z_sb; a.z_st = z_st;
  a.B = B; a.T = T; a.V = V;
  a.tokens = tokens; a.t_sb = t_sb; a.t_st = t_st;
  a.top = stats; a.tot = stats + rows;
  a.slope = {slope, s_sb, s_st};
  a.by = slope_by; a.inv_tau = 1.f / temperature;
  a.up = up; a.unit_done = unit_done;
  a.grad = grad; a.g_sb = g_sb; a.g_st = g_st;
  const int per = ta::GRAD_PIECES * 16 / esize_of(dtype);  // elements of a CTA's piece of a row
  a.chunks = (V + 16 / esize_of(dtype) + per - 1) / per;
  const int64_t items = rows * a.chunks;
  if (items > UINT32_MAX / 2) return fail(TA_ERR_ARG, "%s: too many rows of %d words", who, V);
  a.items = (uint32_t)items;
  // a CTA a piece; where the work is most likely done already, no more of them than the GPU holds
  const unsigned grid = (unsigned)(unit_done ? std::min<int64_t>(items, (int64_t)sm_count() * 6) : items);
  cudaError_t e;
  const cudaStream_t st = S(stream);
  switch (dtype) {
    case TA_F32: e = launch_pdl(ta::logits_grad_kernel<float>, dim3(grid), dim3(ta::GRAD_THREADS), 0, st, a); break;
    case TA_BF16: e = launch_pdl(ta::logits_grad_kernel<__nv_bfloat16>, dim3(grid), dim3(ta::GRAD_THREADS), 0, st, a); break;
    default: e = launch_pdl(ta::logits_grad_kernel<__half>, dim3(grid), dim3(ta::GRAD_THREADS), 0, st, a); break;
  }
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  return TA_OK;
}

}  // extern "C"
