// Gradients of the attention of packed sequences, one translation unit per (element type, head_dim), as
// omni_attn_serving_inst.hip.
#include "omni_attn_serving_bwd_kernel.hpp"

#ifndef OMNI_INST_BF16
#error "compile with -DOMNI_INST_BF16=0|1"
#endif
#ifndef OMNI_INST_D
#error "compile with -DOMNI_INST_D=32|64|128"
#endif

namespace omni_attn {
namespace {

template <auto Kernel>
int launch(const ServeBwdParams& p, unsigned blocks, unsigned threads, size_t lds, hipStream_t stream) {
  static std::atomic<bool> lds_limit_set[kMaxDevices];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return int(e);
  const bool cached = dev >= 0 && dev < kMaxDevices;
  if (!cached || !lds_limit_set[dev].load(std::memory_order_acquire)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
    if (e != hipSuccess) return int(e);
    if (cached) lds_limit_set[dev].store(true, std::memory_order_release);
  }
  ServeBwdParams params = p;
  void* args[] = {&params};
  return int(hipLaunchKernel(reinterpret_cast<const void*>(Kernel), dim3(blocks), dim3(threads), args, lds, stream));
}

}  // namespace

template <bool BF16, int D>
int launch_serve_bwd(const ServeBwdParams& dq, unsigned dq_blocks, const ServeBwdParams& dkdv, unsigned dkdv_blocks, int groups,
                     hipStream_t stream);

// groups: of four waves, that share a tile of keys.
template <>
int launch_serve_bwd<OMNI_INST_BF16 != 0, OMNI_INST_D>(const ServeBwdParams& dq, unsigned dq_blocks, const ServeBwdParams& dkdv,
                                                       unsigned dkdv_blocks, int groups, hipStream_t stream) {
  constexpr bool BF = OMNI_INST_BF16 != 0;
  constexpr int D = OMNI_INST_D;
  const bool cap = dq.s.softcap > 0.f;
  const int e = cap ? launch<serve_dq_kernel<BF, D, true>>(dq, dq_blocks, 256, kServeDqLdsBytes<D>, stream)
                    : launch<serve_dq_kernel<BF, D, false>>(dq, dq_blocks, 256, kServeDqLdsBytes<D>, stream);
  if (e != 0) return e;
  if (groups == 2)
    return cap ? launch<serve_dkdv_kernel<BF, D, true, 2>>(dkdv, dkdv_blocks, 512, kServeDkdvLdsBytes<D, 2>, stream)
               : launch<serve_dkdv_kernel<BF, D, false, 2>>(dkdv, dkdv_blocks, 512, kServeDkdvLdsBytes<D, 2>, stream);
  return cap ? launch<serve_dkdv_kernel<BF, D, true, 1>>(dkdv, dkdv_blocks, 256, kServeDkdvLdsBytes<D, 1>, stream)
             : launch<serve_dkdv_kernel<BF, D, false, 1>>(dkdv, dkdv_blocks, 256, kServeDkdvLdsBytes<D, 1>, stream);
}

}  // namespace omni_attn
