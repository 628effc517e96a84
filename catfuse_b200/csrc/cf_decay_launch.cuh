// cf_decay_launch.cuh — launch templates of the chunk kernel, instantiated per
// element type in cf_decay_tc_{f16,bf16}.cu so that the library builds in parallel.
#pragma once

#include "cf_decay_kernels.cuh"

#include <atomic>

namespace cf {
namespace decayk {

template <typename T, int DK, int DV, bool OUT>
int launch_one(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const DecayArgs& a, int sms,
               cudaStream_t s) {
  using C = Cfg<T, DK, DV, OUT>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  static_assert(C::kColsUsed <= 512, "tensor memory");
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  auto kernel = decay_chunk_kernel<T, DK, DV, OUT>;
  if (dev < 0 || dev >= kMaxDevices || !done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(decay)");
    if (dev >= 0 && dev < kMaxDevices) done[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  const unsigned most = (unsigned)(sms * C::kCtas);
  cfg.gridDim = dim3(a.n_units < most ? a.n_units : most);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  // the set-up overlaps the launch before; tensors are touched only after
  // griddepcontrol.wait
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, q, k, v, a), "decay_attention launch");
}

template <typename T>
int launch_chunks(bool out, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                  const DecayArgs& a, int sms, cudaStream_t s) {
  if (a.Dk <= 64)
    return a.Dv <= 64 ? (out ? launch_one<T, 64, 64, true>(q, k, v, a, sms, s)
                             : launch_one<T, 64, 64, false>(q, k, v, a, sms, s))
                      : (out ? launch_one<T, 64, 128, true>(q, k, v, a, sms, s)
                             : launch_one<T, 64, 128, false>(q, k, v, a, sms, s));
  return a.Dv <= 64 ? (out ? launch_one<T, 128, 64, true>(q, k, v, a, sms, s)
                           : launch_one<T, 128, 64, false>(q, k, v, a, sms, s))
                    : (out ? launch_one<T, 128, 128, true>(q, k, v, a, sms, s)
                           : launch_one<T, 128, 128, false>(q, k, v, a, sms, s));
}

}  // namespace decayk
}  // namespace cf
