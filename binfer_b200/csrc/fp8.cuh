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

// A group's scale, and its reciprocal (off by one place at most).
struct Fp8Scale {
  float s, inv;
};
// ... of a group whose largest size has these bits.  The quotient by 448 is the rounded product with
// 1 / 448 put right by its remainder, which is exact (it equals the division for every significand).
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t largest_bits) {
  Fp8Scale r;
  const float a = __uint_as_float(largest_bits), q = a * (1.f / BF_FP8_MAX);
  r.s = fmaxf(fmaf(fmaf(-q, BF_FP8_MAX, a), 1.f / BF_FP8_MAX, q), 0x1p-100f);
  if (largest_bits >= 0x7f800000u) r.s = __uint_as_float(0x7fffffffu);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inv) : "f"(r.s));
  return r;
}
// the codes of two numbers, the first in the lower byte
__device__ __forceinline__ uint32_t fp8_codes2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// A float that rounds to the code of a / s, for a >= 0.  Codes and the middles between them are among the
// floats of five significant bits; t is the one nearest to a * (1 / s).  A fused multiply-add gives the sign
// of a - t s exactly (t s has 29 bits), and one last place to that side of t decides as the quotient itself
// does: nothing where t is a code, the side where it is a middle, the tie where a / s is t.  (Middles are
// no rarity: of two bfloat16 numbers, the largest and another, the quotient is one every few dozen times.)
__device__ __forceinline__ float fp8_side(float a, const Fp8Scale& k) {
  const uint32_t t = (__float_as_uint(a * k.inv) + 0x40000u) & 0xfff80000u;
  const int side = (int)__float_as_uint(fmaf(-__uint_as_float(t), k.s, a));
  return __uint_as_float(t + (uint32_t)max(min(side, 1), -1));
}
// The codes of N numbers (a multiple of 4), four a word, from their sizes; `signs` has the signs in the
// codes' places.
template <int N>
__device__ __forceinline__ void fp8_codes(const float (&a)[N], const uint32_t (&signs)[N / 4], const Fp8Scale& k,
                                          uint32_t (&c)[N / 4]) {
  const bool finite = k.s == k.s;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint32_t v = fp8_codes2(fp8_side(a[i], k), fp8_side(a[i + 1], k)) |
                       fp8_codes2(fp8_side(a[i + 2], k), fp8_side(a[i + 3], k)) << 16;
    c[i / 4] = finite ? v | (signs[i / 4] & 0x80808080u) : 0x7f7f7f7fu;
  }
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
// Sixteen numbers of a row in the registers' own form, two runs of eight that lie `GAP` apart (8: sixteen
// neighbours; 64: eight lanes' loads and stores of either run are one line each).  `n` numbers are there from
// the first on, counting the gap (the others read as zero); WHOLE: all of them, on 16-byte boundaries.
template <typename T, int GAP>
struct Fp8Sixteen {
  static constexpr int WORDS = (int)sizeof(T) * 4;
  uint32_t w[WORDS];

  template <bool WHOLE>
  __device__ __forceinline__ void load(const T* p, int n) {
    if (WHOLE) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const T* at = i < WORDS / 8 ? p + i * (16 / (int)sizeof(T)) : p + GAP + (i - WORDS / 8) * (16 / (int)sizeof(T));
        const uint4 q = *reinterpret_cast<const uint4*>(at);
        w[4 * i] = q.x;
        w[4 * i + 1] = q.y;
        w[4 * i + 2] = q.z;
        w[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if constexpr (sizeof(T) == 4) {
          const int at = i < 8 ? i : GAP + i - 8;
          w[i] = at < n ? __float_as_uint(p[at]) : 0u;
        } else {
          const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
          const int at = i < 4 ? 2 * i : GAP + 2 * i - 8;
          w[i] = (at < n ? (uint32_t)h[at] : 0u) | (at + 1 < n ? (uint32_t)h[at + 1] << 16 : 0u);
        }
      }
    }
  }
  // the size of a number, and the signs of four
  __device__ __forceinline__ float size(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i] & 0x7fffffffu);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0x7fff0000u : (w[i / 2] & 0x7fffu) << 16);
  }
  __device__ __forceinline__ uint32_t signs(int i) const {            // (of numbers 4 i .., in the bytes' tops)
    if constexpr (sizeof(T) == 4)
      return __byte_perm(__byte_perm(w[4 * i], w[4 * i + 1], 0x0073), __byte_perm(w[4 * i + 2], w[4 * i + 3], 0x0073),
                         0x5410);
    else return __byte_perm(w[2 * i], w[2 * i + 1], 0x7531);
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
    float a[16];
    uint32_t sg[4], c[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] = size(i);
#pragma unroll
    for (int i = 0; i < 4; ++i) sg[i] = signs(i);
    fp8_codes(a, sg, s, c);
    return make_uint4(c[0], c[1], c[2], c[3]);
  }
};
// The factor of a group's sums is the product of two scales.  Scales that are both small or both large have products
// below the floats of full precision, or above all of them, while the product with the sum, of up to 2^25 or down to
// 2^-18, may well be one.  The kernels' loops take such a factor as zero, or as infinity; warps that have the time look
// for them beside (fp8_odd), and the results that they concern are made anew behind the loops (fp8_sum_anew).  (A look
// within the loops, even at one flag a group, cost 2 to 15 % of a product.)
__device__ __forceinline__ float fp8_loop_factor(float sx, float sw) {
  float f;
  asm("mul.ftz.f32 %0, %1, %2;" : "=f"(f) : "f"(sx), "f"(sw));
  return f;
}
// A factor as two: the sum times `before`, and that times `after`, a power of two, within a multiply-add.  Of s1 s2 in
// 2^-175 .. 2^-126 the first lies in 2^-75 .. 2^-26, of 2^128 .. 2^239 in 2^8 .. 2^119, so that its product with the
// sum underflows nowhere and overflows only where the result does.  (Times less than 2^-175 a sum is less than half of
// the smallest float: nothing, as for two groups of zeros.)
struct Fp8Factor {
  float before, after;
};
__device__ __forceinline__ Fp8Factor fp8_factor(float sx, float sw) {
  const float f = sx * sw;
  if (f > 3.4028234663852886e38f) return Fp8Factor{(sx * 0x1p-60f) * (sw * 0x1p-60f), 0x1p120f};
  if (f < 0x1p-126f) {
    const float before = (sx * 0x1p50f) * (sw * 0x1p50f);
    if (before >= 0x1p-75f) return Fp8Factor{before, 0x1p-100f};
  }
  return Fp8Factor{f, 1.f};
}
// FP8_ODD and more for a product that is no positive float of full precision (the only ones that can be odd)
#define FP8_ODD 0x7f000000u
__device__ __forceinline__ uint32_t fp8_note(float f) { return __float_as_uint(f) - 0x00800000u; }
__device__ __forceinline__ bool fp8_odd(float sx, float sw) {
  return fp8_note(sx * sw) >= FP8_ODD && fp8_factor(sx, sw).after != 1.f;
}
