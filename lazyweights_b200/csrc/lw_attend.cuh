// Device-side parts that the attention kernels over the paged cache share: element types, exponentials, 4-D tile loads.
#pragma once
#include <cuda_bf16.h>

#include "lw_device.cuh"
#include "lw_paged.h"

namespace lw {

// 2^x; -inf gives 0
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// In fp16 weights are taken times 2^lift (most), so that small ones are not lost below its 2^-24; not where scores are so large that 32 bits
// have no digits left for it and a weight could round beyond fp16.  `reference`: what scores are taken from, which is what O and l go by.
constexpr float kLiftLimit = 4194304.f;   // 2^22: whole and quarter numbers are exact below
template <typename T>
__device__ __forceinline__ float lift(float reference, float most) {
  return std::is_same<T, __half>::value && fabsf(reference) < kLiftLimit ? most : 0.f;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A box of a 4-D tensor map (no multicast) -> shared memory, its bytes counted on `bar`.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}

}  // namespace lw
