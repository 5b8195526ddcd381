// fp32, fp16 and bf16 values as operands of the bf16 matrix instructions: each
// as a sum of bf16 pieces, products accumulated in fp32.
#pragma once

#include "bm_seq.h"

namespace bm {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

// bf16 pieces of two values, as the halves of a word each
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
template <int N>
__device__ __forceinline__ void split2(uint32_t (&p)[N], float x, float y) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const v2f v = {x, y};
    p[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2bf));
    if (k + 1 < N) {
      x -= __uint_as_float(p[k] << 16);
      y -= __uint_as_float(p[k] & 0xffff0000u);
    }
  }
}
// of eight values, as MFMA operands
template <int N>
__device__ __forceinline__ void split8(v8bf (&p)[N], const float* v) {
  u32x4 w[N];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t q[N];
    split2<N>(q, v[2 * e], v[2 * e + 1]);
#pragma unroll
    for (int k = 0; k < N; ++k) w[k][e] = q[k];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) p[k] = __builtin_bit_cast(v8bf, w[k]);
}

template <typename T>
struct Pieces;  // IN: of an input; Y: of what only y depends on
template <>
struct Pieces<float> {
  static constexpr int IN = 3, Y = 3;
};
template <>
struct Pieces<_Float16> {
  static constexpr int IN = 2, Y = 3;
};
template <>
struct Pieces<__bf16> {
  static constexpr int IN = 1, Y = 2;
};
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane),
                 hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// keeps the compiler from working the offsets of 16 rows out ahead of the
// loop and holding them in registers
__device__ __forceinline__ uint32_t here(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

}  // namespace bm
