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

// The next launch, if it is an overlapped one, may begin and wait for this
// kernel's end: its blocks are then there at once.
__device__ __forceinline__ void let_next_launch_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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

// Elements in 32-bit words, one or two: their values, words of values (rounded
// to nearest), the larger of two words element by element (NaN only where both
// are), and the largest of a word's.
template <typename T> struct Words;
template <> struct Words<float> {
  static constexpr uint32_t kLeast = 0xff800000u; // -infinity
  static __device__ __forceinline__ uint32_t of(float x, float) { return __float_as_uint(x); }
  static __device__ __forceinline__ float value(uint32_t word, int) {
    return __uint_as_float(word);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float largest(uint32_t word) { return __uint_as_float(word); }
};
template <> struct Words<__nv_bfloat16> {
  static constexpr uint32_t kLeast = 0xff80ff80u; // -infinity
  static __device__ __forceinline__ uint32_t of(float low, float high) {
    const auto pair = __floats2bfloat162_rn(low, high);
    uint32_t word;
    memcpy(&word, &pair, 4);
    return word;
  }
  static __device__ __forceinline__ float value(uint32_t word, int half) {
    return __uint_as_float(half == 0 ? word << 16 : word & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    __nv_bfloat162 x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    x = __hmax2(x, y);
    memcpy(&a, &x, 4);
    return a;
  }
  static __device__ __forceinline__ float largest(uint32_t word) {
    return fmaxf(value(word, 0), value(word, 1));
  }
};
template <> struct Words<__half> {
  static constexpr uint32_t kLeast = 0xfc00fc00u; // -infinity
  static __device__ __forceinline__ uint32_t of(float low, float high) {
    const auto pair = __floats2half2_rn(low, high);
    uint32_t word;
    memcpy(&word, &pair, 4);
    return word;
  }
  static __device__ __forceinline__ float value(uint32_t word, int half) {
    __half2 x;
    memcpy(&x, &word, 4);
    return half == 0 ? __low2float(x) : __high2float(x);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    __half2 x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    x = __hmax2(x, y);
    memcpy(&a, &x, 4);
    return a;
  }
  static __device__ __forceinline__ float largest(uint32_t word) {
    return fmaxf(value(word, 0), value(word, 1));
  }
};

// Width neighbouring elements in words (a single 16-bit one in the lower half),
// moved as one access of at most 16 bytes.
template <typename T, int Width> struct WordVector {
  static constexpr int kBytes = Width * static_cast<int>(sizeof(T));
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t at[kWords];

  __device__ __forceinline__ void load(const T *from) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4 *>(from);
      at[0] = v.x;
      at[1] = v.y;
      at[2] = v.z;
      at[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2 *>(from);
      at[0] = v.x;
      at[1] = v.y;
    } else if constexpr (kBytes == 4) {
      at[0] = *reinterpret_cast<const uint32_t *>(from);
    } else {
      at[0] = *reinterpret_cast<const uint16_t *>(from);
    }
  }
  __device__ __forceinline__ void store(T *to) const {
    if constexpr (kBytes == 16) {
      *reinterpret_cast<uint4 *>(to) = make_uint4(at[0], at[1], at[2], at[3]);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2 *>(to) = make_uint2(at[0], at[1]);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t *>(to) = at[0];
    } else {
      *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(at[0]);
    }
  }
};

// 2^x; 0 for -infinity.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t shared_address(const void *pointer) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(pointer));
}

// 16 bytes from global to shared memory; zeros where `valid` is false.
__device__ __forceinline__ void copy_16(uint32_t to, uint64_t from, bool valid) {
  const uint32_t bytes = valid ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void commit_copies() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int Pending> __device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(Pending) : "memory");
}

// Counts a block in, by one thread after a barrier of its threads: what they
// wrote before is seen by the threads that pass a barrier with the one that
// counted in later. Returns how many were there before.
__device__ __forceinline__ uint32_t arrive(uint32_t *counter) {
  uint32_t before;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
               : "=r"(before)
               : "l"(__cvta_generic_to_global(counter))
               : "memory");
  return before;
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

} // namespace lrrt::ops

#endif // LRRT_PAGED_COMMON_CUH_
