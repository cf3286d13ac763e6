// C ABI of the serving operators: the 8-bit paged cache (append, attention) and the verification of drafted tokens.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "../../include/treeattn_b200.h"
#include "host.cuh"
#include "paged.cuh"
#include "paged_tile.cuh"
#include "verify.cuh"

namespace ta_host {
// This translation unit's device error record (see ta_device_error), read and cleared.
cudaError_t paged_device_error(int* out4) {
  cudaError_t e = cudaMemcpyFromSymbol(out4, ta::g_dev_err, 4 * sizeof(int));
  if (e != cudaSuccess || out4[0] == 0) return e;
  const int zero[4] = {0, 0, 0, 0};
  return cudaMemcpyToSymbol(ta::g_dev_err, zero, 4 * sizeof(int));
}
}  // namespace ta_host

namespace {

using namespace ta_host;

// Arguments that describe the cache and the call's rows, shared by the entry points.
int check_cache(const char* who, const void* pool, const void* tail, const int32_t* table, int64_t table_sb, int n_pages,
                int max_pages, int page, int dtype, int B, int Hq, int Hkv, int dh, int n_rows, const int32_t* start,
                const int32_t* pos, int max_new) {
  if (dtype != TA_BF16 && dtype != TA_F16) return fail(TA_ERR_ARG, "%s: bad dtype %d (bfloat16 or float16)", who, dtype);
  if (!valid_dh(dh)) return fail(TA_ERR_ARG, "%s: unsupported head dim %d (16, 32, 64, 128)", who, dh);
  if (page != 16 && page != 32 && page != 64)
    return fail(TA_ERR_ARG, "%s: pages of %d tokens (16, 32 or 64)", who, page);
  if (B < 0 || B > 65535 || Hkv < 1 || Hkv > 4096 || Hq < Hkv || Hq > 65535 || Hq % Hkv != 0 || n_rows < 0 || max_new < 0)
    return fail(TA_ERR_ARG, "%s: bad sizes B=%d Hq=%d Hkv=%d rows=%d max_new=%d (Hq a multiple of Hkv)", who, B, Hq, Hkv,
                n_rows, max_new);
  if (n_pages < 1 || max_pages < 0 || table_sb < max_pages || (int64_t)(max_pages + 1) * page > INT_MAX)
    return fail(TA_ERR_ARG, "%s: bad page counts n_pages=%d max_pages=%d (row stride %lld)", who, n_pages, max_pages,
                (long long)table_sb);
  if (!pool || !tail || !table || !start || !pos) return fail(TA_ERR_ARG, "%s: null pointer", who);
  if (!aligned16(pool) || !aligned16(tail)) return fail(TA_ERR_ARG, "%s: the pool and the tail must be 16-byte aligned", who);
  return TA_OK;
}

template <typename T, int DH>
int run_append(const ta::AppendParams& a, int B, cudaStream_t st) {
  const int64_t spans = (a.max_new - 1) / ta::APPEND_SPAN + 2;  // that one sequence's new tokens can touch
  if (spans * a.c.Hkv > INT_MAX / 2 || (int64_t)a.max_new * a.Hq * DH > INT_MAX)
    return fail(TA_ERR_ARG, "ta_paged_append: too many rows of one sequence in a call");
  ta::AppendParams p = a;
  p.page_ctas = (int)spans * a.c.Hkv;
  int q_ctas = 0;
  if (a.q_out) {  // four 16-byte pieces to a thread, as far as that fills the GPU
    const int64_t work = ((int64_t)a.max_new * a.Hq * (DH / 8) + ta::APPEND_THREADS * 4 - 1) / (ta::APPEND_THREADS * 4);
    q_ctas = (int)std::min<int64_t>(work, std::max(1, sm_count() * 32 / std::max(B, 1)));
  }
  const size_t smem = (size_t)2 * ta::APPEND_SPAN * (DH + 8) * 2;
  const cudaError_t e = launch_pdl(ta::paged_append_kernel<T, DH>, dim3(p.page_ctas + q_ctas, B), dim3(ta::APPEND_THREADS), smem,
                                   st, p);
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "ta_paged_append: launch failed: %s", cudaGetErrorString(e));
  return TA_OK;
}

template <typename T, int DH, int NT>
int run_attn_nt(const ta::AttnParams& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.max_new * (p.Hq / p.c.Hkv);
  const int64_t tiles = (rows + 8 * NT - 1) / (8 * NT);
  if (tiles > INT_MAX) return fail(TA_ERR_ARG, "ta_paged_attn: too many rows");
  static SmemAttr attr;
  constexpr int smem = ta::attn_smem_bytes<DH, NT>();
  if (int r = allow_smem(attr, ta::paged_attn_kernel<T, DH, NT>, smem, "ta_paged_attn")) return r;
  ta::paged_attn_kernel<T, DH, NT><<<dim3((unsigned)tiles, p.c.Hkv, p.B), ta::ATTN_WARPS * 32, smem, st>>>(p);
  return check_launch("ta_paged_attn");
}

// A workspace begins with the arrival counters, one per item, in a place of one size for every call: whatever shapes share a
// workspace, no call's states lie where another's counters are expected to be zero.
constexpr int64_t kItems = 1 << 16;
constexpr int64_t kCounterBytes = kItems * 4;

// The split form: two states for every warp of the grid.
template <int DH, int NT>
int64_t split_bytes() {
  using SH = ta::SplitShape<DH, NT>;
  return kCounterBytes + (int64_t)sm_count() * SH::WARPS * 2 * SH::STATE * 4;
}

template <int DH>
int64_t split_bytes_dh(int64_t rows) {
  if (rows <= 8) return split_bytes<DH, 1>();
  if (rows <= 16) return split_bytes<DH, 2>();
  if (rows <= 24) return split_bytes<DH, 3>();
  return split_bytes<DH, 4>();
}

// Rows of one (sequence, kv head) up to which the call takes the split form (more would not fit its registers). Split / tile form
// in us: 24 rows, 16 sequences of 8000, 4 heads of 64: 37 / 59, of 128: 64 / 92. At 32 rows either may win: one sequence of 30000, 8
// heads of 64: 46 / 72, of 128: 84 / 96; 8 of 30000: 127 / 165, 255 / 292; 16 of 8000, 4 heads: 53 / 60, 98 / 93; 64 of 2000: 62 / 54,
// 108 / 94; 4 of 1000: 23 / 21, 33 / 27; 2 of 20000, 2 heads: 35 / 54, 86 / 68. The lengths, which decide it, are on the device.
constexpr int kSplitRows = 32;

bool split_takes(int64_t B, int64_t Hkv, int64_t rows, int64_t max_pages, int P) {
  return rows <= kSplitRows && B <= ta::SPLIT_MAX_BATCH && B * Hkv <= kItems && B * Hkv * (max_pages * P / 32 + 7) <= INT_MAX;
}

// Whether an item's states are joined late: by the parts it has where the batch is even, and the cache as full as it can be (the
// lengths are on the device). Where they are not, it is the wrong side: one sequence of 4096, 12 heads of 64, in a table for 32768
// takes 11.6 us, in one of its own length 9.5; one of 30000 among 15 of 500, 8 heads, 8 rows, takes 27 us at 64 and 47 at 128, alone
// 18.5 and 29.
template <int DH, int NT>
bool split_late(const ta::AttnParams& p) {
  using SH = ta::SplitShape<DH, NT>;
  const int64_t held = (int64_t)p.c.max_pages * p.c.P;
  const int64_t seen = p.window > 0 ? std::min<int64_t>(held, (int64_t)p.window + p.max_new) : held;
  const int64_t parts = std::min<int64_t>((int64_t)sm_count() * SH::WARPS / ((int64_t)p.B * p.c.Hkv),
                                          seen / (SH::UT * ta::SPLIT_MIN_UNITS));
  return parts * SH::STATE * 4 > ta::SPLIT_SPOT_BYTES;
}

template <typename T, int DH, int NT, bool LATE, bool PROBE = false>
int launch_split(const ta::AttnParams& p, void* ws, int64_t ws_bytes, cudaStream_t st) {
  using SH = ta::SplitShape<DH, NT>;
  const int64_t need = split_bytes<DH, NT>();
  if (!ws || !aligned16(ws) || ws_bytes < need)
    return fail(TA_ERR_ARG, "ta_paged_attn: a workspace of %lld bytes is needed (16-byte aligned; got %lld)", (long long)need,
                (long long)ws_bytes);
  static SmemAttr attr;
  const int smem = SH::RING + SH::BAR_BYTES + 12 * (p.B + 1);
  if (int r = allow_smem(attr, ta::paged_split_kernel<T, DH, NT, LATE, PROBE>, smem, "ta_paged_attn")) return r;
  float* states = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + kCounterBytes);
  const cudaError_t e = launch_pdl(ta::paged_split_kernel<T, DH, NT, LATE, PROBE>, dim3(sm_count()), dim3(SH::WARPS * 32), smem,
                                   st, p, reinterpret_cast<int32_t*>(ws), states);
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "ta_paged_attn: launch failed: %s", cudaGetErrorString(e));
  return TA_OK;
}

template <typename T, int DH, int NT, bool PROBE = false>
int run_split(const ta::AttnParams& p, void* ws, int64_t ws_bytes, cudaStream_t st) {
  if constexpr (ta::split_spot<DH, NT>()) {
    if (!split_late<DH, NT>(p)) return launch_split<T, DH, NT, false, PROBE>(p, ws, ws_bytes, st);
  }
  return launch_split<T, DH, NT, true, PROBE>(p, ws, ws_bytes, st);
}

// The tile form (head dims 64 and 128): CTAs that share a tile's blocks, as many as make the tiles fill the GPU.
int64_t tiles_of(int64_t rows) { return (rows + ta::TILE_ROWS - 1) / ta::TILE_ROWS; }
int tile_splits(int64_t B, int64_t Hkv, int64_t rows, int dh) {
  const int64_t items = B * Hkv * tiles_of(rows), room = (int64_t)sm_count() * (dh == 64 ? 2 : 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>(ta::TILE_MAX_SPLITS, room / std::max<int64_t>(1, items)));
}
int64_t tile_bytes(int64_t B, int64_t Hkv, int64_t rows, int dh) {
  const int splits = tile_splits(B, Hkv, rows, dh);
  if (splits == 1) return 0;
  const int64_t items = B * Hkv * tiles_of(rows);
  return kCounterBytes + items * splits * ta::TILE_ROWS * (dh + 2) * 4;
}

template <typename T, int DH, bool PROBE = false>
int run_tile(const ta::AttnParams& p, int64_t rows, void* ws, int64_t ws_bytes, cudaStream_t st) {
  using C = ta::TileShape<T, DH>;
  const int64_t need = tile_bytes(p.B, p.c.Hkv, rows, DH), tiles = tiles_of(rows);
  if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need))
    return fail(TA_ERR_ARG, "ta_paged_attn: a workspace of %lld bytes is needed (16-byte aligned; got %lld)", (long long)need,
                (long long)ws_bytes);
  ta::TileParams tp{};
  tp.a = p;
  tp.tiles = (int)tiles;
  tp.splits = tile_splits(p.B, p.c.Hkv, rows, DH);
  tp.counters = reinterpret_cast<int32_t*>(ws);
  tp.states = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + kCounterBytes);
  static SmemAttr attr;
  constexpr int smem = 1024 + C::BYTES + (int)sizeof(ta::TileBars);
  if (int r = allow_smem(attr, ta::paged_tile_kernel<T, DH, PROBE>, smem, "ta_paged_attn")) return r;
  const cudaError_t e = launch_pdl(ta::paged_tile_kernel<T, DH, PROBE>, dim3((unsigned)(tiles * tp.splits), p.c.Hkv, p.B),
                                   dim3(ta::TILE_THREADS), smem, st, tp);
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "ta_paged_attn: launch failed: %s", cudaGetErrorString(e));
  return TA_OK;
}

template <typename T, int DH>
int run_attn(const ta::AttnParams& p, void* ws, int64_t ws_bytes, cudaStream_t st) {
  const int64_t rows = (int64_t)p.max_new * (p.Hq / p.c.Hkv);
  if (split_takes(p.B, p.c.Hkv, rows, p.c.max_pages, p.c.P)) {
    if (rows <= 8) return run_split<T, DH, 1>(p, ws, ws_bytes, st);
    if (rows <= 16) return run_split<T, DH, 2>(p, ws, ws_bytes, st);
    if (rows <= 24) return run_split<T, DH, 3>(p, ws, ws_bytes, st);
    return run_split<T, DH, 4>(p, ws, ws_bytes, st);
  }
  if constexpr (DH >= 64) {
    if (rows > kSplitRows) return run_tile<T, DH>(p, rows, ws, ws_bytes, st);
  }
  if (rows <= 8) return run_attn_nt<T, DH, 1>(p, st);
  if (rows <= 16 || DH == 128) return run_attn_nt<T, DH, 2>(p, st);  // 32 rows of head dim 128 do not fit the registers
  return run_attn_nt<T, DH, DH == 128 ? 2 : 4>(p, st);
}

// Clusters of cs CTAs, one per sequence, with programmatic dependent launch.
cudaError_t launch_verify(void (*kern)(ta::VerifyParams), int cs, cudaStream_t st, const ta::VerifyParams& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * cs));
  cfg.blockDim = dim3(ta::VERIFY_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

int paged_attn(const char* who, int probe, const void* pool, const void* tail, const int32_t* table, int64_t table_sb,
               int n_pages, int max_pages, int page, int dtype, int B, int Hq, int Hkv, int dh, const void* q, int64_t q_sr,
               int64_t q_sh, int n_rows, const int32_t* start, const int32_t* pos, int max_new, float scale, int window,
               void* out, int64_t o_sr, int64_t o_sh, float* lse, void* ws, int64_t ws_bytes, void* stream) {
  g_err.clear();
  if (int r = check_cache(who, pool, tail, table, table_sb, n_pages, max_pages, page, dtype, B, Hq, Hkv, dh, n_rows, start,
                          pos, max_new))
    return r;
  if (window < 0) return fail(TA_ERR_ARG, "%s: window %d", who, window);
  if (window >= (int64_t)(max_pages + 1) * page) window = 0;  // longer than any sequence
  if (B == 0 || n_rows == 0 || max_new == 0) return TA_OK;
  if (!q || !out) return fail(TA_ERR_ARG, "%s: null pointer", who);
  if (!rows_aligned(q, 2, {q_sr, q_sh}) || !rows_aligned(out, 2, {o_sr, o_sh}))
    return fail(TA_ERR_ARG, "%s: q and out rows must be 16-byte aligned", who);
  if ((int64_t)max_new * (Hq / Hkv) > INT_MAX / 2) return fail(TA_ERR_ARG, "%s: too many rows", who);
  ta::AttnParams p{};
  p.c = {const_cast<unsigned char*>(reinterpret_cast<const unsigned char*>(pool)), const_cast<void*>(tail), table, table_sb,
         n_pages, max_pages, Hkv, page};
  p.q = q; p.q_sr = q_sr; p.q_sh = q_sh;
  p.start = start; p.pos = pos;
  p.B = B; p.n_rows = n_rows; p.max_new = max_new; p.Hq = Hq;
  p.scale = scale; p.window = window;
  p.out = out; p.o_sr = o_sr; p.o_sh = o_sh; p.lse = lse;
  const cudaStream_t st = S(stream);
  if (probe >= 0) {
    const int64_t rows = (int64_t)max_new * (Hq / Hkv);
    p.probe = probe;
    if (dtype != TA_BF16 || dh != 64 || (rows > 8 && rows <= kSplitRows) || !split_takes(B, Hkv, 1, max_pages, page))
      return fail(TA_ERR_ARG, "%s: bfloat16 rows of head dim 64, at most 8 or more than %d of a kv head", who, kSplitRows);
    if (rows <= 8) return run_split<__nv_bfloat16, 64, 1, true>(p, ws, ws_bytes, st);
    return run_tile<__nv_bfloat16, 64, true>(p, rows, ws, ws_bytes, st);
  }
#define TA_ATTN(T)                                                              \
  switch (dh) {                                                                 \
    case 16: return run_attn<T, 16>(p, ws, ws_bytes, st);                                   \
    case 32: return run_attn<T, 32>(p, ws, ws_bytes, st);                                   \
    case 64: return run_attn<T, 64>(p, ws, ws_bytes, st);                                   \
    default: return run_attn<T, 128>(p, ws, ws_bytes, st);                                  \
  }
  if (dtype == TA_BF16) { TA_ATTN(__nv_bfloat16) } else { TA_ATTN(__half) }
#undef TA_ATTN
}

}  // namespace

extern "C" {

int ta_paged_append(void* pool, void* tail, const int32_t* table, int64_t table_sb, int n_pages, int max_pages, int page,
                    int dtype, int B, int Hkv, int dh, const void* k, const void* v, int64_t k_sr, int64_t k_sh,
                    int64_t v_sr, int64_t v_sh, int n_rows, const int32_t* start, const int32_t* pos, int max_new,
                    const float* cosv, const float* sinv, int n_pos, int rot, const void* q, int Hq, int64_t q_sr,
                    int64_t q_sh, void* q_out, void* stream) {
  g_err.clear();
  const char* who = "ta_paged_append";
  if (!q_out) Hq = Hkv;
  if (int r = check_cache(who, pool, tail, table, table_sb, n_pages, max_pages, page, dtype, B, Hq, Hkv, dh, n_rows, start,
                          pos, max_new))
    return r;
  if (rot < 0 || rot > dh || rot % 2 != 0) return fail(TA_ERR_ARG, "%s: rotated dims %d (even, at most the head dim %d)", who, rot, dh);
  if (B == 0 || n_rows == 0 || max_new == 0) return TA_OK;
  if (!k || !v || (rot && (!cosv || !sinv || n_pos < 1)) || (q_out && !q)) return fail(TA_ERR_ARG, "%s: null pointer", who);
  if (!rows_aligned(k, 2, {k_sr, k_sh}) || !rows_aligned(v, 2, {v_sr, v_sh}))
    return fail(TA_ERR_ARG, "%s: k and v rows must be 16-byte aligned", who);
  if (rot % 16 == 0) {  // pairs by eight: queries and tables are read in 16-byte pieces too (otherwise element by element)
    if (q_out && (!rows_aligned(q, 2, {q_sr, q_sh}) || !aligned16(q_out)))
      return fail(TA_ERR_ARG, "%s: q and q_out rows must be 16-byte aligned", who);
    if (rot && (!aligned16(cosv) || !aligned16(sinv)))
      return fail(TA_ERR_ARG, "%s: the rotation's tables must be 16-byte aligned", who);
  }
  ta::AppendParams p{};
  p.c = {reinterpret_cast<unsigned char*>(pool), tail, table, table_sb, n_pages, max_pages, Hkv, page};
  p.k = k; p.v = v; p.q = q;
  p.k_sr = k_sr; p.k_sh = k_sh; p.v_sr = v_sr; p.v_sh = v_sh; p.q_sr = q_sr; p.q_sh = q_sh;
  p.q_out = q_out;
  p.start = start; p.pos = pos;
  p.cosv = cosv; p.sinv = sinv; p.n_pos = n_pos; p.rot = rot;
  p.n_rows = n_rows; p.max_new = max_new; p.Hq = Hq;
  const cudaStream_t st = S(stream);
#define TA_APPEND(T)                                                              \
  switch (dh) {                                                                   \
    case 16: return run_append<T, 16>(p, B, st);                                  \
    case 32: return run_append<T, 32>(p, B, st);                                  \
    case 64: return run_append<T, 64>(p, B, st);                                  \
    default: return run_append<T, 128>(p, B, st);                                 \
  }
  if (dtype == TA_BF16) { TA_APPEND(__nv_bfloat16) } else { TA_APPEND(__half) }
#undef TA_APPEND
}

int64_t ta_paged_attn_workspace(int B, int Hq, int Hkv, int dh, int max_new) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || max_new < 1 || !valid_dh(dh)) return 0;
  const int64_t rows = (int64_t)max_new * (Hq / Hkv);
  if (rows > kSplitRows) return dh >= 64 ? tile_bytes(B, Hkv, rows, dh) : 0;
  switch (dh) {
    case 16: return split_bytes_dh<16>(rows);
    case 32: return split_bytes_dh<32>(rows);
    case 64: return split_bytes_dh<64>(rows);
    default: return split_bytes_dh<128>(rows);
  }
}

int ta_paged_attn(const void* pool, const void* tail, const int32_t* table, int64_t table_sb, int n_pages, int max_pages,
                  int page, int dtype, int B, int Hq, int Hkv, int dh, const void* q, int64_t q_sr, int64_t q_sh,
                  int n_rows, const int32_t* start, const int32_t* pos, int max_new, float scale, int window, void* out,
                  int64_t o_sr, int64_t o_sh, float* lse, void* ws, int64_t ws_bytes, void* stream) {
  return paged_attn("ta_paged_attn", -1, pool, tail, table, table_sb, n_pages, max_pages, page, dtype, B, Hq, Hkv, dh, q,
                    q_sr, q_sh, n_rows, start, pos, max_new, scale, window, out, o_sr, o_sh, lse, ws, ws_bytes, stream);
}

int ta_paged_attn_probe(int worker, const void* pool, const void* tail, const int32_t* table, int64_t table_sb, int n_pages,
                        int max_pages, int page, int dtype, int B, int Hq, int Hkv, int dh, const void* q, int64_t q_sr,
                        int64_t q_sh, int n_rows, const int32_t* start, const int32_t* pos, int max_new, float scale,
                        int window, void* out, int64_t o_sr, int64_t o_sh, float* lse, void* ws, int64_t ws_bytes,
                        void* stream) {
  g_err.clear();
  if (worker < 0) return fail(TA_ERR_ARG, "ta_paged_attn_probe: worker %d", worker);
  return paged_attn("ta_paged_attn_probe", worker, pool, tail, table, table_sb, n_pages, max_pages, page, dtype, B, Hq, Hkv, dh, q,
                    q_sr, q_sh, n_rows, start, pos, max_new, scale, window, out, o_sr, o_sh, lse, ws, ws_bytes, stream);
}

int ta_verify_drafts(const void* p, int64_t p_sb, int64_t p_sr, const void* q, int64_t q_sb, int64_t q_sr, int dtype, int B,
                     int G, int V, const int64_t* drafts, const float* u, const int32_t* n, int64_t* tokens,
                     int32_t* accepted, void* stream) {
  g_err.clear();
  const char* who = "ta_verify_drafts";
  if (!valid_dtype(dtype)) return fail(TA_ERR_ARG, "%s: bad dtype %d", who, dtype);
  if (B < 0 || B > INT_MAX / 8 || G < 0 || G > 1024 || V < 1 || V > (1 << 24))
    return fail(TA_ERR_ARG, "%s: bad sizes B=%d G=%d V=%d (at most 1024 drafts, 2^24 words)", who, B, G, V);
  if (B == 0) return TA_OK;
  if (!p || !u || !tokens || !accepted || (G && (!q || !drafts))) return fail(TA_ERR_ARG, "%s: null pointer", who);
  ta::VerifyParams a{p, q, p_sb, p_sr, q_sb, q_sr, drafts, u, n, B, G, V, 0, tokens, accepted};
  // CTAs of a sequence: more while the shares stay above 4096 words and all CTAs are resident together (4 an SM)
  int cs = 1;
  while (cs < ta::VERIFY_MAX_CLUSTER && V / (2 * cs) >= 4096 && (int64_t)B * 2 * cs <= 4 * (int64_t)sm_count()) cs *= 2;
  const int step = 32 * 16 / esize_of(dtype), warps = cs * ta::VERIFY_WARPS;
  a.seg = ((V + warps - 1) / warps + step - 1) / step * step;
  const cudaStream_t st = S(stream);
  cudaError_t e;
  switch (dtype) {
    case TA_F32: e = launch_verify(ta::verify_kernel<float>, cs, st, a); break;
    case TA_BF16: e = launch_verify(ta::verify_kernel<__nv_bfloat16>, cs, st, a); break;
    default: e = launch_verify(ta::verify_kernel<__half>, cs, st, a); break;
  }
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  return TA_OK;
}

}  // extern "C"
