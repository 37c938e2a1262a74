// Shared pieces of the training / serving operators (cit_linear.hip,
// cit_policy.hip, cit_gradnorm.hip): element types, loads at any alignment,
// rounding, sums over a wave and a block.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/citadels.h"

typedef __bf16 bf16_t;
typedef _Float16 fp16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes at any address of the element's own alignment: gfx950 loads and
// stores global memory unaligned, so this is one global_load_dwordx4 (rows of
// odd widths cost the lines they straddle, not an instruction per element).
struct __attribute__((packed, aligned(2))) any16 { u32x4 v; };
struct __attribute__((packed, aligned(2))) any8 { uint32_t v[2]; };

__device__ __forceinline__ u32x4 load16(const void* p) { return static_cast<const any16*>(p)->v; }
__device__ __forceinline__ void store16(void* p, u32x4 v) { static_cast<any16*>(p)->v = v; }

template <typename T>
struct Pack16 {                                     // 16 bytes as elements
  static constexpr int N = 16 / sizeof(T);
  union { u32x4 raw; T e[N]; };
};

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }   // round to nearest even

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

// A grid of at least `blocks` workgroups of at most 1,024 threads: a dimension's threads have to be under 2^32, so
// more than 2^21 of them go on in y (those past the last one have nothing to do).
static inline dim3 wide_grid(int64_t blocks) {
  constexpr int64_t MOST = 1 << 21;
  const int64_t y = (blocks + MOST - 1) / MOST;
  return y <= 1 ? dim3((unsigned)blocks) : dim3((unsigned)MOST, (unsigned)y);
}

// The launch's own error, as the other entry points report it.
static inline int launch_status() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}
