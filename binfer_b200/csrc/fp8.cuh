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

// A group's scale, and its reciprocal from below and above.
struct Fp8Scale {
  float s, low, high;
};
// ... of a group whose largest size has these bits.  The quotient by 448 is the rounded product with
// 1 / 448 put right by its remainder, which is exact (it equals the division for every significand).
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t largest_bits) {
  Fp8Scale r;
  const float a = __uint_as_float(largest_bits), q = a * (1.f / BF_FP8_MAX);
  r.s = fmaxf(fmaf(fmaf(-q, BF_FP8_MAX, a), 1.f / BF_FP8_MAX, q), 0x1p-100f);
  if (largest_bits >= 0x7f800000u) r.s = __uint_as_float(0x7fffffffu);
  float inv;                                       // (off by one place at most)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(r.s));
  r.low = inv * (1.f - 0x1p-21f);
  r.high = inv * (1.f + 0x1p-21f);
  return r;
}
// the codes of two quotients, the first in the lower byte
__device__ __forceinline__ uint32_t fp8_codes2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// A float that rounds to the code of x / s: the rounded quotient q; where q lies on the middle of two
// codes and x / s does not, the sign of x - q s, which a fused multiply-add gives exactly (q has five
// bits), says on which side, and one last place to that side decides the rounding.
__device__ __forceinline__ float fp8_quotient(float x, float s) {
  float q = __fdiv_rn(x, s);
  const float r = fmaf(-q, s, x);
  const bool middle = fabsf(q) < 0x1p-6f ? q * 1024.f == rintf(q * 1024.f)
                                         : (__float_as_uint(q) & 0xfffffu) == 0x80000u;
  if (middle && q != 0.f && r != 0.f)
    q = __uint_as_float(__float_as_uint(q) + ((r > 0.f) == (q > 0.f) ? 1u : 0xffffffffu));
  return q;
}
// The codes of four numbers.  x / s lies between x * low and x * high (2^-21 to either side covers the
// three roundings between): where both round to the same code it is that, else (four numbers in 2^14)
// the quotients are taken.
__device__ __forceinline__ uint32_t fp8_codes4(const float* x, const Fp8Scale& k) {
  const uint32_t c = fp8_codes2(x[0] * k.low, x[1] * k.low) | fp8_codes2(x[2] * k.low, x[3] * k.low) << 16;
  const uint32_t d = fp8_codes2(x[0] * k.high, x[1] * k.high) | fp8_codes2(x[2] * k.high, x[3] * k.high) << 16;
  if (c == d) return c;
  return fp8_codes2(fp8_quotient(x[0], k.s), fp8_quotient(x[1], k.s)) |
        fp8_codes2(fp8_quotient(x[2], k.s), fp8_quotient(x[3], k.s)) << 16;
  return c;
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
// Sixteen neighbouring numbers of a row (as many as 32-bit words hold of them are a register), of which
// `n` are there (the others read as zero); WHOLE: all sixteen, on a 16-byte boundary.
template <typename T>
struct Fp8Sixteen {
  static constexpr int WORDS = (int)sizeof(T) * 4;
  uint32_t w[WORDS];

  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* p, int n) {
    if (WHOLE) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = q.x;
        w[4 * i + 1] = q.y;
        w[4 * i + 2] = q.z;
        w[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if constexpr (sizeof(T) == 4) {
          w[i] = i < n ? __float_as_uint(p[i]) : 0u;
        } else {
          const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
          w[i] = (2 * i < n ? (uint32_t)h[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)h[2 * i + 1] << 16 : 0u);
        }
      }
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  // the largest size, as the bits of a float (those of a NaN are above an infinity's)
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
      return max(m << 16, m & 0xffff0000u);
    }
  }
  __device__ __forceinline__ uint4 codes(const Fp8Scale& s) const {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x[4] = {value(4 * i), value(4 * i + 1), value(4 * i + 2), value(4 * i + 3)};
      c[i] = fp8_codes4(x, s);
    }
    return make_uint4(c[0], c[1], c[2], c[3]);
  }
};
// The factor of a group's sums: the product of two scales, held at the largest float, so that a sum of
// zero stays zero where the product alone is out of range.  (NaN stays NaN.)
__device__ __forceinline__ float fp8_factor(float sx, float sw) {
  const float f = sx * sw;
  return f > 3.4028234663852886e38f ? 3.4028234663852886e38f : f;
}
