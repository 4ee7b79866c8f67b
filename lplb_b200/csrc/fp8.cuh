// Values in 8 bits: e4m3 with one power-of-two scale (e8m0: a biased exponent) for every block of
// 128 along a row, the form in which the tensor cores multiply the scales in by themselves.
// The reference holds no values in 8 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace lplb {
namespace fp8 {

constexpr int kBlock = 128;  // values per scale

// Biased exponent of the smallest power of two s with amax / s <= 448, the largest e4m3 value, given
// the bits of amax.  448 is 1.75 * 2^8: with amax = m * 2^e the exponent is e - 8, one more where
// m > 1.75 (the addition carries into the exponent exactly then).  Never below 2^-126, so that both
// the scale and its reciprocal are normal floats; a block of zeros gets that scale.
__host__ __device__ __forceinline__ uint32_t scale_exponent(uint32_t amax_bits) {
  const uint32_t e = (amax_bits + 0x1FFFFFu) >> 23;
  return e > 9u ? e - 8u : 1u;
}
// 2^-(e - 127) for 1 <= e <= 253
__device__ __forceinline__ float reciprocal_of(uint32_t exponent) { return __uint_as_float((254u - exponent) << 23); }

// Bits of |v| for the maximum of a block, 0 where v is not finite: an infinity or NaN does not
// touch its block's scale.
__device__ __forceinline__ uint32_t magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
// Largest magnitude of eight values: fmaxf passes over NaN, and where an infinity was seen the
// finite values are looked through once more.
__device__ __forceinline__ uint32_t magnitude8(const float2 (&v)[4]) {
  float top = fmaxf(fabsf(v[0].x), fabsf(v[0].y));
#pragma unroll
  for (int i = 1; i < 4; ++i) top = fmaxf(fmaxf(top, fabsf(v[i].x)), fabsf(v[i].y));
  if (top < __uint_as_float(0x7F800000u)) return __float_as_uint(top);
  uint32_t finite = 0;  // an infinity, or eight NaN
#pragma unroll
  for (int i = 0; i < 4; ++i) finite = max(finite, max(magnitude(v[i].x), magnitude(v[i].y)));
  return finite;
}
// v / scale for the conversion below: e4m3 has no infinity, so one becomes NaN (v - v) instead of 448.
__device__ __forceinline__ float scaled(float v, float reciprocal) { return fmaf(v, reciprocal, v - v); }
// Two values to e4m3, round to nearest even: off by at most 2^-4 of the value, or half of 2^-9 scales.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// two products, sums, products and sums in 32 bits by one instruction
__device__ __forceinline__ uint64_t bits2(float2 v) { return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ float2 from_bits2(uint64_t b) { return make_float2(__uint_as_float((uint32_t)b), __uint_as_float((uint32_t)(b >> 32))); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return from_bits2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return from_bits2(r);
}
// Eight values times `factor` to e4m3; `finite` is false where one of the eight may be infinite.
__device__ __forceinline__ uint2 pack8(float2 (&v)[4], float factor, bool finite) {
  uint32_t h[4];
  if (!finite) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i].x += v[i].x - v[i].x, v[i].y += v[i].y - v[i].y;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = mul2(v[i], make_float2(factor, factor));
    h[i] = pack2(q.x, q.y);
  }
  return make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
}
__device__ __forceinline__ bool all_finite(const float2 (&v)[4]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(fmaxf(top, fabsf(v[i].x)), fabsf(v[i].y));
  return top < __uint_as_float(0x7F800000u);
}

// ---- eight consecutive values of a row -------------------------------------------------------
// n of them (n <= 0: none) lie inside the row, the others are zero.  VEC: all or none, on a 16-byte boundary.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};
__device__ __forceinline__ void set_zero(float& v) { v = 0.f; }
__device__ __forceinline__ void set_zero(__nv_bfloat16& v) { v = __float2bfloat16_rn(0.f); }
__device__ __forceinline__ void set_zero(__half& v) { v = __float2half_rn(0.f); }

// to and from 32 bits, two values of 16 at a time
template <typename T>
__device__ __forceinline__ void unpack(const Eight<T>& raw, float2 (&f)[4]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4)
      f[i] = make_float2(raw.v[2 * i], raw.v[2 * i + 1]);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>)
      f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    else
      f[i] = __half22float2(*reinterpret_cast<const __half2*>(w + i));
  }
}
template <typename T>
__device__ __forceinline__ Eight<T> pack(const float2 (&f)[4]) {
  Eight<T> raw;
  uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      raw.v[2 * i] = f[i].x;
      raw.v[2 * i + 1] = f[i].y;
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 two = __floats2bfloat162_rn(f[i].x, f[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&two);
    } else {
      const __half2 two = __floats2half2_rn(f[i].x, f[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
  }
  return raw;
}
// a + b, rounded once to their type
template <typename T>
__device__ __forceinline__ Eight<T> add(const Eight<T>& a, const Eight<T>& b) {
  Eight<T> sum;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum.v[i] = a.v[i] + b.v[i];
  } else {
    using Two = std::conditional_t<std::is_same_v<T, __nv_bfloat16>, __nv_bfloat162, __half2>;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<Two*>(&sum)[i] = __hadd2(reinterpret_cast<const Two*>(&a)[i], reinterpret_cast<const Two*>(&b)[i]);
  }
  return sum;
}
template <bool VEC, typename T>
__device__ __forceinline__ Eight<T> load_raw(const T* p, int n) {
  Eight<T> raw;
#pragma unroll
  for (int i = 0; i < 8; ++i) set_zero(raw.v[i]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      if (n > 0) reinterpret_cast<uint4*>(&raw)[i] = ld_behind_wait(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) raw.v[i] = p[i];
  }
  return raw;
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_raw(T* __restrict__ p, int n, const Eight<T>& raw) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      if (n > 0) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&raw)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = raw.v[i];
  }
}
template <bool VEC>
__device__ __forceinline__ void store8_e4m3(uint8_t* p, int n, uint2 q) {
  if constexpr (VEC) {
    if (n > 0) *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}
// Largest value over the 16 lanes (a block of 128, eight values each) that this lane is one of.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

}  // namespace fp8
}  // namespace lplb
