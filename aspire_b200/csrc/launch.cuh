// Host-side launch helpers shared by the extern "C" entry points: launches with
// a programmatic dependency, shared-memory opt-ins and the tensor-map encoder.
#pragma once

#include <atomic>
#include <utility>

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include "../../include/aspire_b200.h"
#include "errors.h"

namespace aspire {

// Launches `kernel` with a programmatic dependency on the preceding work in
// the stream (every kernel begins with griddepcontrol.launch_dependents +
// wait, so it is scheduled early but reads nothing before its predecessor
// has finished).
template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const char* what,
           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), what);
}

// Bound of one pipeline wait of the tcgen05 kernels, in nanoseconds.
uint64_t wait_limit_ns();

inline int current_sm_count(int* out) {
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  return check_cuda(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev),
                    "cudaDeviceGetAttribute(SM count)");
}

// Dynamic shared memory a kernel has been opted in to, per device: the
// attribute set by cudaFuncSetAttribute applies to the current device only,
// so a host thread that drives several GPUs sets it once on each.
constexpr int kMaxDevices = 64;
struct SmemOptIn {
  std::atomic<int> bytes[kMaxDevices];
  SmemOptIn() {
    for (auto& b : bytes) b.store(48 * 1024);
  }
};

// Opt-in to large dynamic shared memory once per (kernel, device, size).
inline int ensure_smem(const void* func, size_t bytes, SmemOptIn& cache) {
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  const bool cached = dev >= 0 && dev < kMaxDevices;
  if (cached && int(bytes) <= cache.bytes[dev].load(std::memory_order_relaxed)) return ASPIRE_OK;
  rc = check_cuda(cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)),
                  "cudaFuncSetAttribute(max dynamic smem)");
  if (rc == ASPIRE_OK && cached) {
    int cur = cache.bytes[dev].load(std::memory_order_relaxed);
    while (cur < int(bytes) && !cache.bytes[dev].compare_exchange_weak(cur, int(bytes))) {
    }
  }
  return rc;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link).
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }
  return fn;
}

}  // namespace aspire
