// Attention of packed sequences, one translation unit per (element type, head_dim): compiled several times with
// -DOMNI_INST_BF16={0,1} -DOMNI_INST_D={32,64,128}; each object defines the kernels of that pair, for packed and paged
// keys, behind one C++ symbol.
#include "omni_attn_serving_kernel.hpp"

#ifndef OMNI_INST_BF16
#error "compile with -DOMNI_INST_BF16=0|1"
#endif
#ifndef OMNI_INST_D
#error "compile with -DOMNI_INST_D=32|64|128"
#endif

namespace omni_attn {
namespace {

template <auto Kernel>
int launch(const ServeParams& p, unsigned blocks, unsigned threads, size_t lds, hipStream_t stream) {
  static std::atomic<bool> lds_limit_set[kMaxDevices];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return int(e);
  const bool cached = dev >= 0 && dev < kMaxDevices;
  if (lds != 0 && (!cached || !lds_limit_set[dev].load(std::memory_order_acquire))) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
    if (e != hipSuccess) return int(e);
    if (cached) lds_limit_set[dev].store(true, std::memory_order_release);
  }
  ServeParams params = p;
  void* args[] = {&params};
  return int(hipLaunchKernel(reinterpret_cast<const void*>(Kernel), dim3(blocks), dim3(threads), args, lds, stream));
}

}  // namespace

template <bool BF16, int D>
int launch_serve(const ServeParams& p, int rows, int waves, unsigned blocks, hipStream_t stream);

// rows, waves: tiles of 128 or 64 rows (these without parts) and four waves, or of 32 rows and one wave or four.
template <>
int launch_serve<OMNI_INST_BF16 != 0, OMNI_INST_D>(const ServeParams& p, int rows, int waves, unsigned blocks, hipStream_t stream) {
  constexpr bool BF = OMNI_INST_BF16 != 0;
  constexpr int D = OMNI_INST_D;
  constexpr size_t few = kFewLdsBytes<D>;
  const Keys keys = p.page_table == nullptr ? kPacked : ((1 << p.page_shift) >= kPageOfStep ? kPages : kSmallPages);
#define OMNI_SERVE(kernel, n, threads, lds)                                                        \
  (keys == kPacked  ? launch<kernel<BF, D, kPacked, n>>(p, blocks, threads, lds, stream)           \
   : keys == kPages ? launch<kernel<BF, D, kPages, n>>(p, blocks, threads, lds, stream)            \
                    : launch<kernel<BF, D, kSmallPages, n>>(p, blocks, threads, lds, stream))
  int e;
  if (rows == 128) {
    e = OMNI_SERVE(serve_tile_kernel, 128, 256, (kTileLdsBytes<D, 128>));
  } else if (rows == 64) {
    e = OMNI_SERVE(serve_tile_kernel, 64, 256, (2 * kTileLdsBytes<D, 64>));
  } else if (waves == 1) {
    e = OMNI_SERVE(serve_few_kernel, 1, 64, few);
  } else {
    e = OMNI_SERVE(serve_few_kernel, 4, 256, 4 * few);
  }
#undef OMNI_SERVE
  if (e != 0 || p.share == 0.f) return e;
  const int64_t joined = int64_t(p.T) * ((p.Hk * p.G + kJoinRows<D> - 1) / kJoinRows<D>);
  const unsigned join_blocks = unsigned((joined + 3) / 4);
  return rows == 128 ? launch<serve_join_kernel<BF, D, 128>>(p, join_blocks, 256, 0, stream)
                     : launch<serve_join_kernel<BF, D, 32>>(p, join_blocks, 256, 0, stream);
}

}  // namespace omni_attn
