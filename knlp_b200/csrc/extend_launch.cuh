// Launches of the two tensor-core extend kernels for a pair of plane modes.
#pragma once

#include <atomic>

#include "extend_few.cuh"

namespace knlp {
namespace extend {

// One pair of plane modes, both head dimensions: the kernel for many rows on `many`, then the one
// for few rows on `few`, each a programmatic dependent of the launch before it.
template <int KM, int VM>
int launch_extend_pair(const Params& many, const Params& few, bool only_few, int grid, cudaStream_t st);

template <auto FN>
int launch_dependent(const Params& p, int grid, int threads, int smem, cudaStream_t st) {
  // the attribute is set once per device (a bit each)
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return KNLP_ERR_NO_DEVICE;
  }
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(FN, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
      cudaGetLastError();
      return KNLP_ERR_NO_DEVICE;
    }
    ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, FN, p) != cudaSuccess) {
    cudaGetLastError();
    return KNLP_ERR_LAUNCH;
  }
  return KNLP_OK;
}

template <int KM, int VM, int D>
int launch_extend_one(const Params& many, const Params& few, bool only_few, int grid, cudaStream_t st) {
  const int rc = only_few ? KNLP_OK : launch_dependent<extend_mma_kernel<KM, VM, D>>(many, grid, kThreads, Layout<KM, VM, D>::kBytes, st);
  if (rc) return rc;
  return launch_dependent<few::extend_few_kernel<KM, VM, D>>(few, grid, few::kFewThreads, few::FewLayout<KM, VM, D>::kBytes, st);
}

#define KNLP_EXTEND_PAIR(KM, VM)                                                              \
  namespace knlp {                                                                            \
  namespace extend {                                                                          \
  template <>                                                                                 \
  int launch_extend_pair<KM, VM>(const Params& many, const Params& few, bool only_few,        \
                                 int grid, cudaStream_t st) {                                 \
    return many.a.head_dim == 64 ? launch_extend_one<KM, VM, 64>(many, few, only_few, grid, st)   \
                                 : launch_extend_one<KM, VM, 128>(many, few, only_few, grid, st); \
  }                                                                                           \
  }                                                                                           \
  }

}  // namespace extend
}  // namespace knlp
