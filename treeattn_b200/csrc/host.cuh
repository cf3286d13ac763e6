// Host-side helpers of the C entry points: the failure message, launch checks, alignment checks, per-device launch
// settings and the programmatic dependent launch. Shared by the library's translation units.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <string>
#include <utility>

#include "../../include/treeattn_b200.h"

namespace ta_host {

inline thread_local std::string g_err;

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_err = buf;
  return code;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(TA_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return TA_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// a row of dh elements of `esize` bytes read in 16-byte chunks: base and every stride must keep 16-byte
// alignment
inline bool rows_aligned(const void* base, int esize, std::initializer_list<int64_t> strides) {
  if (!aligned16(base)) return false;
  for (int64_t s : strides)
    if ((s * esize) % 16 != 0) return false;
  return true;
}

inline int esize_of(int dtype) { return dtype == TA_F32 ? 4 : 2; }

inline bool valid_dtype(int dtype) { return dtype == TA_F32 || dtype == TA_BF16 || dtype == TA_F16; }

inline bool valid_dh(int dh) { return dh == 16 || dh == 32 || dh == 64 || dh == 128; }

inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }

// Per-device state of one launcher. cudaFuncSetAttribute and the occupancy and SM-count queries answer for the
// current device only, so a process that drives several GPUs keeps one entry per device (the first 64 devices
// are cached; others are asked again on every call).
constexpr int kDevCache = 64;

inline int current_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  return dev;
}

// SMs of the current device (148 where there is none to ask).
inline int sm_count() {
  static std::atomic<int> have[kDevCache];
  const int dev = current_device();
  const bool cached = dev >= 0 && dev < kDevCache;
  if (cached) {
    const int n = have[dev].load(std::memory_order_relaxed);
    if (n > 0) return n;
  }
  int n = 0;
  if (dev < 0 || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 148;
  }
  if (cached) have[dev].store(n, std::memory_order_relaxed);
  return n;
}

// The dynamic shared-memory size a call site has allowed for its kernel, per device (0 = not yet).
struct SmemAttr {
  std::atomic<size_t> bytes[kDevCache];
};

// Allow `bytes` of dynamic shared memory for kern on the current device. The attribute is always set to the most
// the device gives one block beside the kernel's static shared memory: a kernel launched from several call sites
// (or launcher instantiations) then never has its limit lowered by one of them under another's launch.
template <typename K>
int allow_smem(SmemAttr& a, K* kern, size_t bytes, const char* what) {
  const int dev = current_device();
  const bool cached = dev >= 0 && dev < kDevCache;
  if (cached) {
    const size_t have = a.bytes[dev].load(std::memory_order_relaxed);
    if (have >= bytes) return TA_OK;
    if (have != 0) return fail(TA_ERR_ARG, "%s: %zu B of dynamic shared memory, above the %zu B a block can have",
                               what, bytes, have);
  }
  int optin = 0;
  cudaFuncAttributes fa;
  if (cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev < 0 ? 0 : dev) != cudaSuccess ||
      cudaFuncGetAttributes(&fa, kern) != cudaSuccess)
    return check_launch(what);
  const size_t most = (size_t)optin > fa.sharedSizeBytes ? (size_t)optin - fa.sharedSizeBytes : 0;
  if (bytes > most)
    return fail(TA_ERR_ARG, "%s: %zu B of dynamic shared memory, above the %zu B a block can have", what, bytes, most);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) {
    const cudaError_t e = cudaGetLastError();
    return fail(TA_ERR_CUDA, "%s: dynamic shared memory limit of %zu B refused: %s", what, most, cudaGetErrorString(e));
  }
  if (cached) a.bytes[dev].store(most, std::memory_order_relaxed);
  return TA_OK;
}

// Launch with programmatic stream serialization: the kernel may start while the previous kernel of the stream is
// still running (it calls griddepcontrol.wait before reading anything that kernel writes).
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace ta_host
