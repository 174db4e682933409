// Host helpers shared by the launchers: pointer alignment, the device's SM count
// and the dynamic shared memory limit of a kernel, each looked up or set once.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <mutex>

namespace ecah {

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool aligned16(const void* p) { return aligned_to(p, 16); }

// SM count of the current device, looked up once per device; 0 without one.
inline int device_sms() {
  constexpr int kMaxDev = 64;
  static int cache[kMaxDev] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return 0;
  if (cache[dev] > 0) return cache[dev];
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  cache[dev] = sms;
  return sms;
}

// cudaFuncSetAttribute once per (kernel, device, value): the attribute is a
// property of the kernel on a device, so later launches skip the call.
// forget_smem drops the remembered values (a launch that failed sets them
// again: after cudaDeviceReset the kernels come back without them).
struct SmemMemo {
  static constexpr int kSlots = 128;
  std::mutex mu;
  const void* fn[kSlots];
  int dev[kSlots], val[kSlots];
  int used = 0;
};

inline SmemMemo& smem_memo() {
  static SmemMemo m;
  return m;
}

inline void forget_smem() {
  try {
    SmemMemo& m = smem_memo();
    std::lock_guard<std::mutex> lock(m.mu);
    m.used = 0;
  } catch (...) {                      // no exception leaves a C entry point
  }
}

inline cudaError_t remember_smem(const void* fn, int smem) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  SmemMemo& m = smem_memo();
  std::lock_guard<std::mutex> lock(m.mu);
  for (int i = 0; i < m.used; ++i)
    if (m.fn[i] == fn && m.dev[i] == dev && m.val[i] >= smem) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  for (int i = 0; i < m.used; ++i)
    if (m.fn[i] == fn && m.dev[i] == dev) { m.val[i] = smem; return cudaSuccess; }
  if (m.used < SmemMemo::kSlots) {
    m.fn[m.used] = fn; m.dev[m.used] = dev; m.val[m.used] = smem; ++m.used;
  }
  return cudaSuccess;
}

template <typename Args>
inline cudaError_t set_smem_once(void (*kernel)(const Args), int smem) {
  try {
    return remember_smem(reinterpret_cast<const void*>(kernel), smem);
  } catch (...) {
    return cudaErrorUnknown;
  }
}

// Launches `fn` with `smem` bytes of dynamic shared memory, setting the limit
// first where it may exceed the 48 KB default beside static shared memory; one retry
// with the limit set afresh.  The launch may begin while the kernel before it in the
// stream ends (programmatic stream serialisation): `fn` calls grid_start() before its
// first access to global memory.
template <typename Args>
inline bool launch_kernel(void (*fn)(const Args), dim3 grid, int threads, int smem, cudaStream_t s, const Args& args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int attempt = 0; attempt < 2; ++attempt) {
    if (smem > 32 * 1024 && set_smem_once(fn, smem) != cudaSuccess) { cudaGetLastError(); return false; }
    if (cudaLaunchKernelEx(&cfg, fn, args) == cudaSuccess) return true;
    cudaGetLastError();
    forget_smem();
  }
  return false;
}

}  // namespace ecah
