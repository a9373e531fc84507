// Device helpers that the kernels of llm_kernels.h share.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "llm_kernels.h"

namespace om {
namespace llm {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// N neighbouring elements of a tensor, as they lie in memory: aligned to the
// largest power of two that divides their size, 16 bytes at most.
template <typename T, int N>
struct alignas(((sizeof(T) * N) & -(sizeof(T) * N)) < 16 ? ((sizeof(T) * N) & -(sizeof(T) * N))
                                                          : 16) Pack {
  T v[N];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) {
  return __builtin_bit_cast(
      float, (unsigned)__builtin_bit_cast(unsigned short, x) << 16);
}
// Results leave with one rounding, to nearest even.
template <typename T> __device__ __forceinline__ T from_f32(float x) {
  return (T)x;
}

// The largest value among the 16 lanes of a row of the wave (lanes 16 i ..
// 16 i + 15), in every lane: four rotations within the row.
__device__ __forceinline__ float row_max(float v) {
#define OM_ROW_STEP(ctrl)                                                      \
  v = __builtin_fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(  \
                             0, __builtin_bit_cast(int, v), ctrl, 0xF, 0xF,      \
                             true)))
  OM_ROW_STEP(0x128); // row_ror:8
  OM_ROW_STEP(0x124);
  OM_ROW_STEP(0x122);
  OM_ROW_STEP(0x121);
#undef OM_ROW_STEP
  return v;
}

// Consecutive blocks go round-robin to the 8 XCDs, each with an L2 of its own:
// renumbered so that an XCD gets a contiguous range of `n` blocks.
__device__ __forceinline__ int xcd_contiguous(int id, int n) {
  const int per = n >> 3;
  return per > 0 && id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

} // namespace llm
} // namespace om
