// Host-side pieces that every entry point uses: the driver's tensor-map encoder, per-kernel preparation and the
// launch itself.
#pragma once
#include "../../include/fa4_nvfp4.h"

#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <atomic>
#include <map>
#include <mutex>
#include <utility>

namespace fa4 {

constexpr uint64_t kDefaultBudgetNs = 2000ull * 1000 * 1000;
// SMs of a B200, for rules that must give one answer on the host alone (the size of a workspace is asked for
// without a device) and for the shares of the streaming kernels; persistent grids ask the device.
constexpr int64_t kSms = 148;

inline PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) ==
            cudaSuccess &&
        qres == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    }
  });
  return fn;
}

// Byte tensor of rank 4, innermost dimension contiguous; box = {box0, box1, box2, box3} bytes /
// rows; 64-byte swizzle when the innermost box is 64 bytes.
inline bool encode_u8_4d(CUtensorMap* m, const void* base, const uint64_t (&dims)[4],
                  const uint64_t (&strides)[3], const uint32_t (&box)[4], CUtensorMapSwizzle sw) {
  auto fn = get_encode();
  if (fn == nullptr) return false;
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides,
                        box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

// Launch epoch recorded with a device-side failure (see ptx.cuh): launches modulo 256.
inline uint32_t next_launch_epoch() {
  static std::atomic<uint32_t> counter{0};
  return counter.fetch_add(1, std::memory_order_relaxed) & 0xffu;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Per-kernel launch preparation, done once per (kernel, device) and remembered: the opt-in to
// `smem_bytes` of dynamic shared memory, the carve-out (see launch_pdl) and -- for the warp-specialised kernels, which re-partition
// registers with setmaxnreg -- the check that the build kept the register count the budget in the
// source assumes (an increase blocks for ever when the CTA was launched with fewer registers per
// thread; such a build is refused with -FA4_E_BUILD instead of being launched).
// expected_regs = 0: no register check.
inline int prepare_kernel(const void* kernel, uint32_t smem_bytes, int expected_regs) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, int> seen;   // -> result of the first preparation
  int dev = 0;
  const cudaError_t ge = cudaGetDevice(&dev);
  if (ge != cudaSuccess) return (int)ge;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_pair(kernel, dev);
  const auto it = seen.find(key);
  if (it != seen.end()) return it->second;
  int rc = 0;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return (int)e;          // not remembered: the caller may retry
  if (expected_regs > 0) {
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) return (int)e;
    if (attr.numRegs < expected_regs) rc = -FA4_E_BUILD;
  }
  seen[key] = rc;
  return rc;
}
template <class Kernel>
int ensure_smem(Kernel kernel, uint32_t bytes) {
  return prepare_kernel(reinterpret_cast<const void*>(kernel), bytes, 0);
}
template <class Kernel>
int ensure_kernel(Kernel kernel, uint32_t bytes, int expected_regs) {
  return prepare_kernel(reinterpret_cast<const void*>(kernel), bytes, expected_regs);
}

// Launch as a programmatic dependent of whatever precedes it in the stream (see pdl_wait in
// ptx.cuh): launch latency and set-up overlap the end of the kernel before.
// Every kernel asks for the largest shared-memory carve-out, also those that use none: an SM changes
// its carve-out only while it is empty, which would take the overlap away again.
template <class... KArgs, class... Args>
int launch_pdl_cluster(unsigned cluster, void (*kernel)(KArgs...), dim3 grid, unsigned threads, uint32_t smem,
                       cudaStream_t stream, Args&&... args) {
  if (int e = prepare_kernel(reinterpret_cast<const void*>(kernel), smem, 0)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
template <class Kernel, class... Args>
int launch_pdl(Kernel kernel, dim3 grid, unsigned threads, uint32_t smem, cudaStream_t stream, Args&&... args) {
  return launch_pdl_cluster(1, kernel, grid, threads, smem, stream, std::forward<Args>(args)...);
}

}  // namespace fa4
