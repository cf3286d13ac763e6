// C ABI of the low-rank adapters beside a shared projection.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/treeattn_b200.h"
#include "adapters.cuh"
#include "host.cuh"

namespace ta_host {
// This translation unit's device error record (see ta_device_error), read and cleared.
cudaError_t adapters_device_error(int* out4) {
  cudaError_t e = cudaMemcpyFromSymbol(out4, ta::g_dev_err, 4 * sizeof(int));
  if (e != cudaSuccess || out4[0] == 0) return e;
  const int zero[4] = {0, 0, 0, 0};
  return cudaMemcpyToSymbol(ta::g_dev_err, zero, 4 * sizeof(int));
}
}  // namespace ta_host

namespace {

using namespace ta_host;

constexpr int FUSED_ROWS = 16;  // rows of one sequence up to which a call takes one kernel, and t need not be kept

int check(const char* who, int dtype, int n_adapters, int K, int N, int r, int n_rows, int B, int max_new, const void* start,
          const void* which) {
  if (dtype != TA_BF16 && dtype != TA_F16) return fail(TA_ERR_ARG, "%s: bad dtype %d (bfloat16 or float16)", who, dtype);
  if (r < 8 || r > 128 || r % 8 != 0) return fail(TA_ERR_ARG, "%s: rank %d (a multiple of 8 up to 128)", who, r);
  if (K < 8 || N < 8 || K % 8 != 0 || N % 8 != 0 || K > (1 << 24) || N > (1 << 24))
    return fail(TA_ERR_ARG, "%s: rows of %d and %d columns (multiples of 8)", who, K, N);
  if (n_adapters < 1 || n_adapters > 65535 || n_rows < 0 || n_rows > (1 << 30) || B < 0 || B > 65534 || max_new < 0)
    return fail(TA_ERR_ARG, "%s: bad sizes adapters=%d rows=%d B=%d max_new=%d", who, n_adapters, n_rows, B, max_new);
  if (!start || (B && !which)) return fail(TA_ERR_ARG, "%s: null pointer", who);
  return TA_OK;
}

// Clusters of cs CTAs along x, with programmatic dependent launch.
template <typename P>
int launch(const char* who, void (*kern)(P), SmemAttr& attr, int smem, dim3 grid, int cs, cudaStream_t st, const P& p) {
  if (int r = allow_smem(attr, kern, smem, who)) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(ta::ADAPTER_THREADS);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  return TA_OK;
}

// CTAs of a tile: as many as fill the GPU with one wave of `on_sm` CTAs an SM, each with at least `keep` stages of columns.
int cluster_size(int64_t items, int on_sm, int stages, int keep) {
  int cs = 1;
  while (cs < 8 && items * (cs + 1) <= (int64_t)sm_count() * on_sm && (cs + 1) * keep <= stages) ++cs;
  return cs;
}

template <typename T, int RP>
int run_fused(const char* who, ta::AdapterParams& p, int max_new, cudaStream_t st) {
  using S = ta::AdapterShape<RP>;
  static SmemAttr attr;
  p.tiles = std::max(1, (int)(((int64_t)std::min(max_new, p.n_rows) + 15) / 16));
  // (64 rows of 768 -> 2304, rank 16, on the device: 8.8 us with 8 CTAs a tile, four on an SM, 7.6 with 4; one row of 2048 -> 2048 5.1 with 8,
  // 6.0 with 4)
  const int cs = cluster_size((int64_t)p.tiles * p.B, RP <= 64 ? 2 : 1, (std::max(p.K, p.N) + S::KC - 1) / S::KC, 1);
  const dim3 grid((unsigned)(p.tiles * cs), p.B + (p.out == p.y ? 0 : 1));
  return launch(who, ta::adapter_kernel<T, RP>, attr, S::BYTES, grid, cs, st, p);
}

template <typename T, int RP, bool TRANS>
int run_shrink(const char* who, ta::AdapterParams& p, int max_new, cudaStream_t st) {
  using S = ta::ShrinkShape<RP>;
  static SmemAttr attr;
  if (p.B == 0) return TA_OK;
  p.tiles = std::max(1, (int)(((int64_t)std::min(max_new, p.n_rows) + S::ROWS - 1) / S::ROWS));
  const int cs = cluster_size((int64_t)p.tiles * p.B, RP == 16 ? 4 : RP == 32 ? 3 : 2, (p.K + 32 * S::KS - 1) / (32 * S::KS), 1);
  return launch(who, ta::adapter_shrink_kernel<T, RP, TRANS>, attr, S::BYTES, dim3((unsigned)(p.tiles * cs), p.B), cs, st, p);
}

template <typename T, int RP, bool TRANS>
int run_expand(const char* who, ta::AdapterParams& p, int max_new, cudaStream_t st) {
  using S = ta::ExpandShape<RP, TRANS>;
  static SmemAttr attr;
  p.tiles = std::max(1, (int)(((int64_t)std::min(max_new, p.n_rows) + ta::EXPAND_ROWS - 1) / ta::EXPAND_ROWS));
  const int64_t x = (int64_t)p.tiles * ((p.N + ta::EXPAND_COLS - 1) / ta::EXPAND_COLS);
  if (x > INT_MAX) return fail(TA_ERR_ARG, "%s: too many rows", who);
  const dim3 grid((unsigned)x, p.B + (p.out == p.y ? 0 : 1));
  if (grid.y == 0) return TA_OK;
  return launch(who, ta::adapter_expand_kernel<T, RP, TRANS>, attr, S::BYTES, grid, 1, st, p);
}

// By the rank, filled up to 16, 32, 64 or 128.
#define TA_BY_RANK(F, ...)                  \
  (p.r <= 16   ? F<T, 16 __VA_ARGS__>(who, p, max_new, st) \
   : p.r <= 32 ? F<T, 32 __VA_ARGS__>(who, p, max_new, st) \
   : p.r <= 64 ? F<T, 64 __VA_ARGS__>(who, p, max_new, st) \
               : F<T, 128 __VA_ARGS__>(who, p, max_new, st))

template <typename T>
int run_add(const char* who, ta::AdapterParams& p, int max_new, cudaStream_t st) {
  if (max_new <= FUSED_ROWS) return TA_BY_RANK(run_fused);
  if (int e = TA_BY_RANK(run_shrink, , false)) return e;
  return TA_BY_RANK(run_expand, , false);
}

int run_bwd(const char* who, ta::AdapterParams& p, int max_new, cudaStream_t st) {
  using T = __nv_bfloat16;
  if (int e = TA_BY_RANK(run_shrink, , true)) return e;
  return p.out ? TA_BY_RANK(run_expand, , true) : TA_OK;
}
#undef TA_BY_RANK

template <int RP>
int run_grad(const char* who, const ta::AdapterGradParams& p, cudaStream_t st) {
  using S = ta::AdapterGradShape<RP>;
  static SmemAttr attr;
  const int tiles = (p.da ? (p.K + S::MC - 1) / S::MC : 0) + (p.db ? (p.N + S::MC - 1) / S::MC : 0);
  const dim3 grid(tiles, p.n_adapters, (p.r + S::RT - 1) / S::RT);
  // (a CTA's eight warps take 128 rows at a time)
  const int cs = cluster_size((int64_t)tiles * grid.y * grid.z, 2, (p.n_rows + 127) / 128, 1);
  return launch(who, ta::adapter_grad_kernel<__nv_bfloat16, RP>, attr, S::BYTES, dim3(tiles * cs, grid.y, grid.z), cs, st, p);
}

}  // namespace

extern "C" {

int ta_adapter_add(const void* y, int64_t y_sr, const void* x, int64_t x_sr, const void* a, const void* b, const float* scale,
                   int dtype, int n_adapters, int K, int N, int r, int n_rows, const int32_t* start, const int32_t* which, int B,
                   int max_new, void* out, int64_t o_sr, void* t, void* stream) {
  g_err.clear();
  const char* who = "ta_adapter_add";
  if (int e = check(who, dtype, n_adapters, K, N, r, n_rows, B, max_new, start, which)) return e;
  if (n_rows == 0) return TA_OK;
  if (!x || !y || !a || !b || !out) return fail(TA_ERR_ARG, "%s: null pointer", who);
  if (!rows_aligned(x, 2, {x_sr}) || !rows_aligned(y, 2, {y_sr}) || !rows_aligned(out, 2, {o_sr}) || !aligned16(a) || !aligned16(b))
    return fail(TA_ERR_ARG, "%s: rows and factors must be 16-byte aligned", who);
  if (max_new > FUSED_ROWS && (!t || !aligned16(t)))
    return fail(TA_ERR_ARG, "%s: where a sequence may have more than %d rows t is needed (16-byte aligned)", who, FUSED_ROWS);
  if (out == y && o_sr != y_sr) return fail(TA_ERR_ARG, "%s: out in y's place with other strides", who);
  ta::AdapterParams p{};
  p.x = x; p.y = y; p.out = out;
  p.x_sr = x_sr; p.y_sr = y_sr; p.o_sr = o_sr;
  p.u = a; p.v = b; p.scale = scale;
  p.start = start; p.which = which;
  p.n_rows = n_rows; p.B = B; p.K = K; p.N = N; p.r = r; p.n_adapters = n_adapters;
  p.t = t;
  p.t_by = reinterpret_cast<float*>(reinterpret_cast<char*>(t) + (int64_t)n_rows * r * 4);
  if (B == 0 && out == y) return TA_OK;
  if (dtype == TA_BF16) return run_add<__nv_bfloat16>(who, p, max_new, S(stream));
  return run_add<__half>(who, p, max_new, S(stream));
}

int ta_adapter_bwd(const void* dy, int64_t d_sr, const void* x, int64_t x_sr, const void* a, const void* b, const float* scale,
                   int n_adapters, int K, int N, int r, int n_rows, const int32_t* start, const int32_t* which, int B, int max_new,
                   const void* t, void* u, void* dx, int64_t dx_sr, void* da, void* db, void* stream) {
  g_err.clear();
  const char* who = "ta_adapter_bwd";
  if (int e = check(who, TA_BF16, n_adapters, K, N, r, n_rows, B, max_new, start, which)) return e;
  if (n_rows && (!dy || (da && !x) || (db && !t) || ((dx || da) && (!a || !b || !u))))
    return fail(TA_ERR_ARG, "%s: null pointer", who);
  if (!rows_aligned(dy, 2, {d_sr}) || (da && !rows_aligned(x, 2, {x_sr})) || (dx && !rows_aligned(dx, 2, {dx_sr})) || !aligned16(a) ||
      !aligned16(b) || !aligned16(t) || !aligned16(u) || !aligned16(da) || !aligned16(db))
    return fail(TA_ERR_ARG, "%s: rows and factors must be 16-byte aligned", who);
  const cudaStream_t st = S(stream);
  if ((dx || da) && n_rows > 0) {  // u = s dy B, dx = u A: the forward's kernels with the factors' other sides
    ta::AdapterParams p{};
    p.x = dy; p.x_sr = d_sr;
    p.out = dx; p.o_sr = dx_sr;
    p.u = b; p.v = a; p.scale = scale;
    p.start = start; p.which = which;
    p.n_rows = n_rows; p.B = B; p.K = N; p.N = K; p.r = r; p.n_adapters = n_adapters;
    p.t = u;
    if (int e = run_bwd(who, p, max_new, st)) return e;
  }
  if (!da && !db) return TA_OK;
  ta::AdapterGradParams p{};
  p.x = x; p.dy = dy; p.x_sr = x_sr; p.d_sr = d_sr;
  p.t = t; p.u = u; p.da = da; p.db = db;
  p.start = start; p.which = which;
  p.n_rows = n_rows; p.B = n_rows ? B : 0; p.K = K; p.N = N; p.r = r; p.n_adapters = n_adapters;
  if (r <= 16) return run_grad<16>(who, p, st);
  if (r <= 32) return run_grad<32>(who, p, st);
  if (r <= 64) return run_grad<64>(who, p, st);
  return run_grad<128>(who, p, st);
}

}  // extern "C"
