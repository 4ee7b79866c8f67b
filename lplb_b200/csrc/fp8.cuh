// Values in 8 bits: e4m3 with one power-of-two scale (e8m0: a biased exponent) for every block of
// 128 along a row, the form in which the tensor cores multiply the scales in by themselves.
// The reference holds no values in 8 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

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
// v / scale for the conversion below: e4m3 has no infinity, so one becomes NaN (v - v) instead of 448.
__device__ __forceinline__ float scaled(float v, float reciprocal) { return fmaf(v, reciprocal, v - v); }
// Two values to e4m3, round to nearest even: off by at most 2^-4 of the value, or half of 2^-9 scales.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float reciprocal) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = pack2(scaled(v[2 * i], reciprocal), scaled(v[2 * i + 1], reciprocal));
  return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// ---- eight consecutive values of a row -------------------------------------------------------
// `vec`: the row starts on a 16-byte boundary and p + 8 lies inside it; else up to n (0 to 8) values
// are read one by one and the rest is zero.
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T>
struct alignas(16) Eight {
  T v[8];
};

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, bool vec, int n, float (&f)[8]) {
  if (vec) {
    Eight<T> raw;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<uint4*>(&raw)[0] = __ldg(reinterpret_cast<const uint4*>(p));
      reinterpret_cast<uint4*>(&raw)[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    } else {
      reinterpret_cast<uint4*>(&raw)[0] = __ldg(reinterpret_cast<const uint4*>(p));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_float(raw.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? to_float(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, bool vec, int n, const float (&f)[8]) {
  if (vec) {
    Eight<T> raw;
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.v[i] = from_float<T>(f[i]);
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<const uint4*>(&raw)[0];
    if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<const uint4*>(&raw)[1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_float<T>(f[i]);
  }
}
__device__ __forceinline__ void store8_e4m3(uint8_t* p, bool vec, int n, uint2 q) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = q;
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
