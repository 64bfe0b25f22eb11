// Numbers held in 8 bits: e4m3 codes (1 sign, 4 exponent, 3 fraction bits, largest 448) times a float
// scale that 128 neighbouring numbers of a row share, or a block of 128 x 128 of a weight.
//
// With a the largest size in such a group: s = max(float(a / 448), 2^-100); the code of x is the e4m3
// value nearest to x / s, ties to even, of the quotient itself and not of a float near it (below).  A
// group that holds an infinity or a NaN has the scale NaN.
//
// The lower bound on s keeps every number that the rounding needs in float's normal range: with
// s >= 2^-100 a multiple of 2^-123, the middle of two codes (a multiple of 2^-10 of at most five bits)
// times s is a multiple of 2^-133, so whether x lies above it is decided without underflow.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"

#define BF_FP8_GROUP 128
#define BF_FP8_MAX 448.f

// the scale of a group whose largest size has these bits
__device__ __forceinline__ float fp8_scale(uint32_t largest_bits) {
  if (largest_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  return fmaxf(__fdiv_rn(__uint_as_float(largest_bits), BF_FP8_MAX), 0x1p-100f);
}
// A float that rounds to the code of x / s.  q = x * (1 / s) is off by less than 8 of its last places,
// so it stands unless it is that near to the middle of two codes (one number in 2^15, and those below
// 2^-6, whose codes lie 2^-9 apart).  Else q is the rounded quotient: where it lies on a middle and the
// quotient itself does not, the sign of x - q s, which a fused multiply-add gives exactly (q has five
// bits), says on which side; one last place to that side decides the rounding.
__device__ __forceinline__ float fp8_quotient(float x, float s, float inv) {
  float q = x * inv;
  const uint32_t off = (__float_as_uint(q) + 8u) & 0xfffffu;
  if ((off >= 0x80000u && off <= 0x80010u) || (fabsf(q) < 0x1p-6f && q != 0.f)) {
    q = __fdiv_rn(x, s);
    const float r = fmaf(-q, s, x);
    const bool middle = fabsf(q) < 0x1p-6f ? q * 1024.f == rintf(q * 1024.f)
                                           : (__float_as_uint(q) & 0xfffffu) == 0x80000u;
    if (middle && q != 0.f && r != 0.f)
      q = __uint_as_float(__float_as_uint(q) + ((r > 0.f) == (q > 0.f) ? 1u : 0xffffffffu));
  }
  return q;
}
// the codes of two quotients, the first in the lower byte
__device__ __forceinline__ uint32_t fp8_codes2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t fp8_codes4(const float* x, float s, float inv) {
  return fp8_codes2(fp8_quotient(x[0], s, inv), fp8_quotient(x[1], s, inv)) |
         fp8_codes2(fp8_quotient(x[2], s, inv), fp8_quotient(x[3], s, inv)) << 16;
}
// the values of four codes
__device__ __forceinline__ void fp8_values4(uint32_t codes, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// Eight neighbouring numbers of a row, of which `n` are there (the others read as zero); VEC: the
// address is on a 16-byte boundary and all eight are there.
template <bool VEC>
__device__ __forceinline__ void fp8_load8(const __nv_bfloat16* p, int n, float* v) {
  if (VEC) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t* w = &raw.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void fp8_load8(const float* p, int n, float* v) {
  if (VEC) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}
// the largest size of eight numbers, as bits (those of a NaN are above an infinity's)
__device__ __forceinline__ uint32_t fp8_largest8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
// The factor of a group's sums: the product of two scales, held at the largest float, so that a sum of
// zero stays zero where the product alone is out of range.  (NaN stays NaN.)
__device__ __forceinline__ float fp8_factor(float sx, float sw) {
  const float f = sx * sw;
  return f > 3.4028234663852886e38f ? 3.4028234663852886e38f : f;
}
