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

// N x 4 bytes of elements, moved and taken apart as 32-bit words: structs of 16-bit floats are copied member by
// member, which costs a load or a permutation per element.
template <int N>
struct alignas(N * 4) Words {
  uint32_t w[N];
};
using Words4 = Words<4>;

// Elements 2q and 2q + 1 of packed words as fp32, and back (round to nearest even).
template <typename T, int N>
B2R_DI float2 up_pair(const Words<N>& v, int q)
{
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(v.w[q] << 16), __uint_as_float(v.w[q] & 0xffff0000u));
  } else if constexpr (std::is_same<T, __half>::value) {
    __half2 h;
    memcpy(&h, &v.w[q], 4);
    return __half22float2(h);
  } else {
    return make_float2(__uint_as_float(v.w[2 * q]), __uint_as_float(v.w[2 * q + 1]));
  }
}
template <typename T, int N>
B2R_DI void down_pair(Words<N>& v, int q, float2 f)
{
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    memcpy(&v.w[q], &h, 4);
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    memcpy(&v.w[q], &h, 4);
  } else {
    v.w[2 * q]     = __float_as_uint(f.x);
    v.w[2 * q + 1] = __float_as_uint(f.y);
  }
}
// The bits of element e (compile-time e), and their place in the words.
template <typename T, int N>
B2R_DI void put_bits(Words<N>& v, int e, T x)
{
  if constexpr (sizeof(T) == 2) {
    uint16_t b;
    memcpy(&b, &x, 2);
    v.w[e / 2] = (e & 1) ? ((v.w[e / 2] & 0xffffu) | (uint32_t(b) << 16)) : ((v.w[e / 2] & 0xffff0000u) | b);
  } else {
    memcpy(&v.w[e], &x, 4);
  }
}
template <typename T, int N>
B2R_DI T get_bits(const Words<N>& v, int e)
{
  T x;
  if constexpr (sizeof(T) == 2) {
    const uint16_t b = uint16_t((e & 1) ? v.w[e / 2] >> 16 : v.w[e / 2]);
    memcpy(&x, &b, 2);
  } else {
    memcpy(&x, &v.w[e], 4);
  }
  return x;
}

// V consecutive elements in memory (V x sizeof(T) = 2 ... 32 bytes, aligned to that) and in fp32.
template <typename T, int V>
struct Elems {
  static constexpr int kBytes = V * int(sizeof(T));
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  Words<kWords> v;

  B2R_DI void load(const T* p)
  {
    if constexpr (kBytes >= 4)
      v = *reinterpret_cast<const Words<kWords>*>(p);
    else
      v.w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  // for data that is read once and not written while the kernel runs
  B2R_DI void load_once(const T* p)
  {
    if constexpr (kBytes == 2) {
      uint16_t a;
      asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(a) : "l"(p));
      v.w[0] = a;
    } else {
      const VecOf<uint32_t, kWords> r = load_stream<uint32_t, kWords>(reinterpret_cast<const uint32_t*>(p));
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        v.w[i] = r.e[i];
    }
  }
  B2R_DI void store(T* p) const
  {
    if constexpr (kBytes >= 4)
      *reinterpret_cast<Words<kWords>*>(p) = v;
    else
      *reinterpret_cast<uint16_t*>(p) = uint16_t(v.w[0]);
  }
  B2R_DI void up(float (&f)[V]) const
  {
    if constexpr (V == 1) {
      f[0] = FloatIo<T>::up(get_bits<T>(v, 0));
    } else {
#pragma unroll
      for (int q = 0; q < V / 2; ++q) {
        const float2 x = up_pair<T>(v, q);
        f[2 * q]       = x.x;
        f[2 * q + 1]   = x.y;
      }
    }
  }
  B2R_DI void down(const float (&f)[V])
  {
    if constexpr (V == 1) {
      v.w[0] = 0;
      put_bits<T>(v, 0, FloatIo<T>::down(f[0]));
    } else {
#pragma unroll
      for (int q = 0; q < V / 2; ++q)
        down_pair<T>(v, q, make_float2(f[2 * q], f[2 * q + 1]));
    }
  }
};

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
