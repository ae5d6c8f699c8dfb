// Building blocks of the kernels along the vocabulary axis (embedding.cuh, topk_distill.cuh, sample_tokens.cuh):
// 16-byte vectors of 32- or 16-bit floating-point elements, converted to fp32 and back, and rows that start on
// any element boundary.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

#include <initializer_list>

namespace raft_b200 {
namespace detail {

template <typename T>
struct FloatIo;

template <>
struct FloatIo<float> {
  B2R_DI static float up(float v) { return v; }
  B2R_DI static float down(float v) { return v; }
};
template <>
struct FloatIo<__half> {
  B2R_DI static float up(__half v) { return __half2float(v); }
  B2R_DI static __half down(float v) { return __float2half_rn(v); }
};
template <>
struct FloatIo<__nv_bfloat16> {
  B2R_DI static float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  B2R_DI static __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// elements of T in 16 bytes
template <typename T>
struct Vec16Of {
  static constexpr int value = 16 / int(sizeof(T));
};

// Stores of V consecutive elements, V x sizeof(T) = 2..16 bytes, by one instruction.
template <typename T, int V>
B2R_DI void store_vec(T* p, const VecOf<T, V>& v)
{
  constexpr int bytes = int(sizeof(T)) * V;
  if constexpr (bytes == 16) {
    uint4 w;
    memcpy(&w, &v, 16);
    *reinterpret_cast<uint4*>(p) = w;
  } else if constexpr (bytes == 8) {
    uint2 w;
    memcpy(&w, &v, 8);
    *reinterpret_cast<uint2*>(p) = w;
  } else if constexpr (bytes == 4) {
    uint32_t w;
    memcpy(&w, &v, 4);
    *reinterpret_cast<uint32_t*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      p[i] = v.e[i];
  }
}

// The widest power of two, at most 32, that divides every address and stride given (in bytes).
inline int common_alignment(std::initializer_list<uintptr_t> values)
{
  uintptr_t all = 32;
  for (uintptr_t v : values)
    all |= v;
  return int(all & (~all + 1));
}

}  // namespace detail
}  // namespace raft_b200
