// Attention over the paged cache, in the simplest form: a block per query row and head, a warp per position.
#include <cuda_bf16.h>

#include "lw_device.cuh"
#include "lw_paged.h"

namespace lw {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int kSimpleWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32) k_attend_simple(const __grid_constant__ AttendArgs A) {
  __shared__ int s_seq;
  __shared__ float s_m[kSimpleWarps], s_l[kSimpleWarps], s_o[kSimpleWarps][128];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_seq = -1;
  __syncthreads();
  if (!A.seq.starts) {
    if (threadIdx.x == 0 && row < A.seq.n) s_seq = row;
  } else {
    for (int b = threadIdx.x; b < A.seq.n; b += blockDim.x)
      if (A.seq.starts[b] <= row && row < A.seq.starts[b + 1]) s_seq = b;
  }
  __syncthreads();
  const int b = s_seq, Dh = A.pool.Dh;
  if (b < 0) return;   // a row behind the last sequence
  const long long cap = static_cast<long long>(A.seq.table_cols) * A.pool.page_size;
  int len = max(A.seq.lens[b], 0);
  if (len > cap) {
    if (threadIdx.x == 0) atomicOr(A.err, kErrWordIndex);
    len = static_cast<int>(cap);
  }
  const int last = A.seq.starts ? len - (min(A.seq.starts[b + 1], A.rows) - row) : len - 1;   // the row's position
  const int first = A.window > 0 ? max(0, last - A.window + 1) : 0;
  const T* q = static_cast<const T*>(A.q) + row * A.q_token + head * A.q_head;
  const int kh = head / (A.H / A.pool.Hk);
  float qr[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < 4; ++i) qr[i] = lane + 32 * i < Dh ? to_float(q[lane + 32 * i]) : 0.f;
  for (int p = first + warp; p <= last; p += kSimpleWarps) {
    const int page = A.seq.table[b * A.seq.table_stride + p / A.pool.page_size];
    const bool ok = page >= 0 && page < A.pool.n_pages;
    if (!ok && lane == 0) atomicOr(A.err, kErrWordIndex);
    const long long at = ok ? page * A.pool.page_stride + kh * A.pool.head_stride + (p % A.pool.page_size) * A.pool.token_stride : 0;
    const T *k = static_cast<const T*>(A.pool.k) + at, *v = static_cast<const T*>(A.pool.v) + at;
    float s = 0.f;
    for (int i = 0; i < 4; ++i)
      if (ok && lane + 32 * i < Dh) s = fmaf(qr[i], to_float(k[lane + 32 * i]), s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= A.scale;
    const float m2 = fmaxf(m, s), keep = __expf(m - m2), w = __expf(s - m2);
    m = m2;
    l = l * keep + w;
    for (int i = 0; i < 4; ++i) o[i] = o[i] * keep + (ok && lane + 32 * i < Dh ? w * to_float(v[lane + 32 * i]) : 0.f);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  for (int i = 0; i < 4; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < kSimpleWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int d = threadIdx.x; d < Dh; d += blockDim.x) {
    float sum = 0.f;
    total = 0.f;
    for (int w = 0; w < kSimpleWarps; ++w) {
      const float f = s_l[w] != 0.f ? __expf(s_m[w] - top) : 0.f;
      total += s_l[w] * f;
      sum += s_o[w][d] * f;
    }
    static_cast<T*>(A.out)[row * A.out_token + head * A.out_head + d] = from_float<T>(last < first ? 0.f : sum / total);   // nothing in sight: zeros
  }
}

int launch_attend(ElemType type, const AttendArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.rows, a.H);
  cfg.blockDim = dim3(kSimpleWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, type == kF16 ? k_attend_simple<__half> : k_attend_simple<__nv_bfloat16>, a);
  return note_launch("k_attend_simple");
}

}  // namespace lw
