// Records of the paged cache moved inside their buffers: rec[dst_i] = rec[src_i] for all i at once, in every layer's buffer by one
// launch. The pages of a pool (compaction) and the open pages of sequences (forks of a prompt, beams that take over one
// another's slots) are such records.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <exception>
#include <utility>
#include <vector>

#include "../../include/treeattn_b200.h"
#include "common.cuh"
#include "host.cuh"

namespace {

using namespace ta_host;

// Every thread owns 16 bytes of a record, the same ones in all records of a group, and takes the group's moves in the host's
// order: a record is written only after all moves that read it. So the moves of a group, chains and cycles among them,
// need no second buffer and no barrier, and groups have no record in common (one that is only read apart).
//   move (s, d):  s >= 0 a record to read, SAME the value of the move before, SAVED the one that was saved;
//                 d >= 0 a record to write, SAVE: kept for the end of a cycle, NONE: nothing
// Bound by bytes; four moves' loads are in flight a thread, and a record that several moves read in a row is read once. 12 layers:
// 683 pages of 98 KB moved in 248 us (6.5 TB/s of reads and writes), one sequence's 393 KB into 63 slots in 48 us (6.3 TB/s), six moves among
// eight slots in 13 us, launch and one round of memory.
// The moves travel as the launch's parameters: nothing is uploaded, and a captured call holds its own.
constexpr int THREADS = 256;
constexpr int BATCH = 4;
constexpr int MAX_BUFS = 64;
constexpr int SAME = -1, SAVED = -2;
constexpr int NONE = -1, SAVE = -2;

struct Move {
  int32_t s, d;
};

template <int CAP>
struct Moves {
  char* buf[MAX_BUFS];
  int64_t bytes;                    // of a record
  int columns;                      // bytes / 16
  uint16_t first[CAP / BATCH + 2];  // a group's first batch
  Move m[CAP];
};

template <int CAP>
__global__ void __launch_bounds__(THREADS) record_copy_kernel(const __grid_constant__ Moves<CAP> a) {
  const int col = blockIdx.x * THREADS + threadIdx.x;
  ta::pdl_wait();
  ta::pdl_launch_dependents();
  if (col >= a.columns) return;
  char* const base = a.buf[blockIdx.z] + (int64_t)col * 16;
  const int b1 = a.first[blockIdx.y + 1];
  uint4 last = make_uint4(0u, 0u, 0u, 0u), saved = last;
  for (int b = a.first[blockIdx.y]; b < b1; ++b) {
    const Move* const m = a.m + b * BATCH;
    uint4 v[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (m[u].s >= 0) v[u] = *reinterpret_cast<const uint4*>(base + m[u].s * a.bytes);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (m[u].s >= 0) last = v[u];
      if (m[u].s == SAVED) last = saved;
      if (m[u].d == SAVE) saved = last;
      if (m[u].d >= 0) *reinterpret_cast<uint4*>(base + m[u].d * a.bytes) = last;
    }
  }
}

// The moves in an order that needs no second buffer, group by group; a group begins with a record to read.
struct Plan {
  std::vector<Move> m;
  std::vector<int> first;  // of each group
  std::vector<int> ring;   // where a group's cycle begins (it is the group's end), or past the end
  int source = NONE;       // of the newest move
  void open() {
    first.push_back((int)m.size());
    ring.push_back(INT_MAX);
  }
  void add(int s, int d) {
    const bool fresh = !first.empty() && (int)m.size() == first.back();
    const int before = fresh ? NONE : source;
    m.push_back({s >= 0 && s == before ? SAME : s, d});
    source = s;
  }
};

// Moves whose destinations nobody reads are independent: sorted by source, a batch to a group. The others form trees and cycles of
// "is overwritten by": each is a group, taken from its ends, a cycle opened by saving one record.
int make_plan(Plan& p, const int32_t* src, const int32_t* dst, int n, int n_records) {
  // who writes a record: a table of them all, or the sorted destinations where there are many records to few moves
  const bool dense = n_records <= 65536;
  std::vector<int> by_dst(dense ? n_records : 0, -1);
  std::vector<std::pair<int, int>> sorted;
  for (int i = 0; i < n; ++i) {
    if (src[i] < 0 || src[i] >= n_records || dst[i] < 0 || dst[i] >= n_records)
      return fail(TA_ERR_ARG, "ta_record_copy: move %d from record %d to %d of %d", i, src[i], dst[i], n_records);
    if (!dense) {
      sorted.emplace_back(dst[i], i);
      continue;
    }
    if (by_dst[dst[i]] >= 0) return fail(TA_ERR_ARG, "ta_record_copy: record %d is written twice", dst[i]);
    by_dst[dst[i]] = i;
  }
  std::sort(sorted.begin(), sorted.end());
  for (size_t i = 1; i < sorted.size(); ++i)
    if (sorted[i].first == sorted[i - 1].first)
      return fail(TA_ERR_ARG, "ta_record_copy: record %d is written twice", sorted[i].first);
  auto writer = [&](int record) {
    if (dense) return by_dst[record];
    const auto it = std::lower_bound(sorted.begin(), sorted.end(), std::make_pair(record, -1));
    return it != sorted.end() && it->first == record ? it->second : -1;
  };
  // next[i]: the move that overwrites what move i reads; it waits for i
  std::vector<int> next(n, -1), waits(n, 0), alone, bound;
  for (int i = 0; i < n; ++i)
    if (src[i] != dst[i]) {
      const int w = writer(src[i]);
      if (w >= 0 && src[w] != dst[w]) {
        next[i] = w;
        ++waits[w];
      }
    }
  for (int i = 0; i < n; ++i)
    if (src[i] != dst[i]) (next[i] < 0 && waits[i] == 0 ? alone : bound).push_back(i);
  // those that read one record follow one another
  bool again = false;
  std::vector<char> seen(dense ? n_records : 0, 0);
  if (dense)
    for (int i : alone) {
      again |= seen[src[i]] != 0;
      seen[src[i]] = 1;
    }
  if (again || !dense) std::stable_sort(alone.begin(), alone.end(), [&](int x, int y) { return src[x] < src[y]; });
  for (size_t i = 0; i < alone.size(); ++i) {
    if (i % BATCH == 0) p.open();
    p.add(src[alone[i]], dst[alone[i]]);
  }
  if (bound.empty()) return TA_OK;
  // components: each has one root, or one cycle
  std::vector<int> root(n, -1), order, cycle;
  for (int i : bound) {
    std::vector<int> path;
    int j = i;
    while (j >= 0 && root[j] == -1) {
      root[j] = -2 - i;  // on the walk from i
      path.push_back(j);
      if (next[j] < 0) break;
      j = next[j];
    }
    const int end = j >= 0 && root[j] >= 0 ? root[j] : j;  // a known root, this walk's last move, or the cycle that it met
    for (int k : path) root[k] = end;
  }
  std::vector<std::vector<int>> part(n);
  for (int i : bound) part[root[i]].push_back(i);
  for (int r : bound) {
    if (part[r].empty()) continue;
    p.open();
    order.clear();
    for (int i : part[r])
      if (waits[i] == 0) order.push_back(i);
    for (size_t k = 0; k < order.size(); ++k) {
      const int i = order[k], w = next[i];
      p.add(src[i], dst[i]);
      waits[i] = -1;
      if (w >= 0 && --waits[w] == 0) order.push_back(w);
    }
    // what still waits is a cycle: cycle[k] reads what cycle[k + 1] overwrites. What cycle[0] reads is saved, and goes to its place last
    int c = -1;
    for (int i : part[r])
      if (waits[i] > 0) c = i;
    if (c < 0) continue;
    cycle.clear();
    for (int i = c;;) {
      cycle.push_back(i);
      i = next[i];
      if (i == c) break;
    }
    p.ring.back() = (int)p.m.size();
    p.add(src[cycle[0]], SAVE);
    for (size_t k = 1; k < cycle.size(); ++k) p.add(src[cycle[k]], dst[cycle[k]]);
    p.add(SAVED, dst[cycle[0]]);
  }
  return TA_OK;
}

// The groups of the next launch, from group g and its move `at` on: their number.
template <int CAP>
int pack(const Plan& p, int& g, int& at, Moves<CAP>& a) {
  const int groups = (int)p.first.size();
  int n = 0, slots = 0;
  while (g < groups && slots < CAP) {
    const int end = g + 1 < groups ? p.first[g + 1] : (int)p.m.size(), left = end - at;
    if ((left + BATCH - 1) / BATCH * BATCH > CAP - slots && n > 0) break;  // it begins the next launch
    int take = std::min(left, CAP - slots);  // a group longer than a launch is cut, but not in its cycle: what that saves is in registers
    if (take < left && p.ring[g] < at + take) take = p.ring[g] - at;
    a.first[n++] = (uint16_t)(slots / BATCH);
    std::copy_n(p.m.begin() + at, take, a.m + slots);
    for (int i = at; a.m[slots].s == SAME; --i) a.m[slots].s = p.m[i - 1].s;  // the value of a move in the launch before
    slots += take;
    while (slots % BATCH) a.m[slots++] = {SAME, NONE};
    at += take;
    if (at < end) break;
    ++g;
  }
  a.first[n] = (uint16_t)(slots / BATCH);
  return n;
}

template <int CAP>
int launch(const Plan& p, void* const* bufs, int n_bufs, int64_t bytes, cudaStream_t st) {
  Moves<CAP> a;
  a.bytes = bytes;
  a.columns = (int)(bytes / 16);
  for (int g = 0, at = 0; g < (int)p.first.size();) {
    const int n = pack(p, g, at, a);
    for (int b = 0; b < n_bufs; b += MAX_BUFS) {
      const int nb = std::min(MAX_BUFS, n_bufs - b);
      for (int i = 0; i < nb; ++i) a.buf[i] = reinterpret_cast<char*>(bufs[b + i]);
      const dim3 grid((a.columns + THREADS - 1) / THREADS, n, nb);
      const cudaError_t e = launch_pdl(record_copy_kernel<CAP>, grid, dim3(THREADS), 0, st, a);
      if (e != cudaSuccess) return fail(TA_ERR_CUDA, "ta_record_copy: launch failed: %s", cudaGetErrorString(e));
    }
  }
  return TA_OK;
}

}  // namespace

extern "C" int ta_record_copy(void* const* bufs, int n_bufs, int64_t record_bytes, int n_records, const int32_t* src,
                              const int32_t* dst, int n, void* stream) {
  g_err.clear();
  const char* who = "ta_record_copy";
  if (n_bufs < 0 || n_records < 0 || n < 0 || record_bytes < 16 || record_bytes % 16 != 0 || record_bytes / 16 > INT_MAX / 2)
    return fail(TA_ERR_ARG, "%s: bad sizes: %d buffers, %d records of %lld bytes (a multiple of 16), %d moves", who, n_bufs,
                n_records, (long long)record_bytes, n);
  if (n_bufs == 0 || n == 0) return TA_OK;
  if (!bufs || !src || !dst) return fail(TA_ERR_ARG, "%s: null pointer", who);
  try {
    std::vector<uintptr_t> at(n_bufs);
    for (int i = 0; i < n_bufs; ++i) {
      if (!bufs[i]) return fail(TA_ERR_ARG, "%s: null pointer", who);
      if (!aligned16(bufs[i])) return fail(TA_ERR_ARG, "%s: buffers must be 16-byte aligned", who);
      at[i] = reinterpret_cast<uintptr_t>(bufs[i]);
    }
    std::sort(at.begin(), at.end());
    for (int i = 1; i < n_bufs; ++i)
      if ((int64_t)(at[i] - at[i - 1]) / record_bytes < n_records)
        return fail(TA_ERR_ARG, "%s: two of the buffers overlap", who);
    Plan p;
    if (int r = make_plan(p, src, dst, n, n_records)) return r;
    for (size_t g = 0; g < p.first.size(); ++g) {
      const int64_t end = g + 1 < p.first.size() ? p.first[g + 1] : (int64_t)p.m.size();
      if (end - p.ring[g] > 2048) return fail(TA_ERR_ARG, "%s: a cycle of %d moves (at most 2047)", who, (int)(end - p.ring[g] - 1));
    }
    if (p.m.empty()) return TA_OK;
    const int64_t need = (int64_t)p.m.size() + (BATCH - 1) * (int64_t)p.first.size();
    // parameters of a launch: 1 KB or 17 KB of them
    if (need <= 64) return launch<64>(p, bufs, n_bufs, record_bytes, S(stream));
    return launch<2048>(p, bufs, n_bufs, record_bytes, S(stream));
  } catch (const std::exception& e) {
    return fail(TA_ERR_ARG, "%s: %s", who, e.what());
  }
}
