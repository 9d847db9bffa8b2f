// Launches of the attention kernels: function attributes set once per device, and
// programmatic dependent launch.
#pragma once

#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <utility>

#include "common.cuh"
#include "ptx.cuh"

namespace grinqh {

// Allows `kern` its dynamic shared memory, once per device.
inline int allow_smem(const void* kern, std::atomic<uint64_t>& done, size_t bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return set_error(GRINQH_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  return GRINQH_OK;
}

// How long a wait within an attention kernel lasts before it is lost: GRINQH_ATTENTION_WAIT_US
// microseconds (read on every call), by default 2 s; with 0 all are lost.
inline uint64_t attention_wait_ns() {
  const char* e = std::getenv("GRINQH_ATTENTION_WAIT_US");
  return e ? (uint64_t)std::max(0ll, std::min(std::atoll(e), 2000000ll)) * 1000 : kWaitNs;
}

// SMs of the current device (148 without one).
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      return 148;
    }
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

// A launch that may start while the kernel before it on the stream ends: `kern` must wait
// (wait_prior_grid) before it reads or writes any memory that others do.
template <typename... P, typename... A>
int launch_dependent(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const char* what,
                     A&&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
  if (e != cudaSuccess) return set_error(GRINQH_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace grinqh
