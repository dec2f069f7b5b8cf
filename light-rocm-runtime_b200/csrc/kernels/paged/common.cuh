// Element types and small device helpers of the paged-cache operators.
#ifndef LRRT_PAGED_COMMON_CUH_
#define LRRT_PAGED_COMMON_CUH_

#include "lrrt/ops/kernels.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace lrrt::ops {

constexpr unsigned kAllLanes = 0xffffffffu;

// Launches are overlapped (programmatic dependent): a kernel may start while
// the one before it drains, and reads and writes nothing before this.
__device__ __forceinline__ void wait_for_previous_launch() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <> __device__ __forceinline__ __half from_float<__half>(float x) {
  return __float2half_rn(x);
}

// `Count` elements moved as one load or store of at most 16 bytes.
template <typename T, int Count> struct alignas(sizeof(T) * Count) Vector {
  T at[Count];
};

// 2^x; 0 for -infinity.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

} // namespace lrrt::ops

#endif // LRRT_PAGED_COMMON_CUH_
