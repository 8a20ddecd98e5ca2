// The rotation of a pair by its position's cosine and sine, shared by the rotary and
// the cache-append kernels.
#pragma once

#include "common.hpp"

namespace sm {

// (a, b) -> (a c - b s, b c + a s), every product and sum rounded to f32 by itself: with
// products fused into the sums the result would depend on which of the two the compiler
// fused, and a cache code at a rounding border with it.
__device__ inline void rotate_pair(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
  const float x = a * c - b * s;
  const float y = b * c + a * s;
  a = x;
  b = y;
}

// Eight consecutive values of a row <-> f32. T: float, uint16_t (bf16 bits), _Float16.
template <typename T>
__device__ inline void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, _Float16)) {
        const h2 x = as_h2(v[i]);
        f[2 * i] = (float)x[0];
        f[2 * i + 1] = (float)x[1];
      } else {
        f[2 * i] = bf16lo(v[i]);
        f[2 * i + 1] = bf16hi(v[i]);
      }
    }
  }
}
template <typename T>
__device__ inline uint32_t round2(float a, float b) {
  if constexpr (__is_same(T, _Float16)) {
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
  } else {
    return pack_bf16x2(a, b);
  }
}
template <typename T>
__device__ inline void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = float4{f[0], f[1], f[2], f[3]};
    reinterpret_cast<float4*>(p)[1] = float4{f[4], f[5], f[6], f[7]};
  } else {
    *reinterpret_cast<u32x4*>(p) = u32x4{round2<T>(f[0], f[1]), round2<T>(f[2], f[3]),
                                         round2<T>(f[4], f[5]), round2<T>(f[6], f[7])};
  }
}

// (cos, sin) of N consecutive pairs at table row `pos`; NaN outside the table, which has a
// row at least. (Values are chosen, and one row is always read: stores on two paths would
// keep c and s in memory.)
template <int N>
__device__ inline void load_angles(const float* table, int64_t table_rows, int half, int64_t pos,
                                   int pair, float (&c)[N], float (&s)[N]) {
  const bool in = pos >= 0 && pos < table_rows;
  const float4* p = reinterpret_cast<const float4*>(table + ((in ? pos : 0) * half + pair) * 2);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float4 v = p[i];
    c[2 * i] = in ? v.x : NAN;
    s[2 * i] = in ? v.y : NAN;
    c[2 * i + 1] = in ? v.z : NAN;
    s[2 * i + 1] = in ? v.w : NAN;
  }
}

}  // namespace sm
