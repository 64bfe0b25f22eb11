// The layout of key/value pages held in 4 bits.
//
// A cache of one layer is uint8 [pages][kv_heads][page_size / 8][9 d]: a record of 9 d bytes holds
// eight tokens of one kv head.  Every KV4_GROUP = 64 numbers of a key or value row share a scale s
// and a lowest value m (bfloat16 each); a number is m + s c with a code c of 0 to 15, two codes a
// byte, the lower one in the low half.  Inside a record:
//
//   keys' codes     8 tokens x d / 2 bytes   token after token; a row is four parts of d / 8 bytes, part
//                                            q holds numbers 16 q .. 16 q + 15 of every group
//   values' codes   8 parts x 8 tokens x d / 16 bytes   part r holds numbers 8 r .. 8 r + 7 of every group
//   keys' (s, m)    8 tokens x d / 64 pairs
//   values' (s, m)  the same
//
// so that lane 4 r + q of a warp finds what it needs as a tensor-core operand side by side: its part of
// key r, and its part of the values of tokens 2 q and 2 q + 1.  4.5 bits a number.
#pragma once
#include <cuda_bf16.h>

#define KV4_GROUP 64
#define KV4_EIGHTH 8                       // tokens of a record

// Loaded keys and queries are fp16, which holds a number below 2^-14 to 2^-25 only.  A key or query off by that moves a
// score by 2^-25 / sqrt(3) times the other's length times the scale: at this scale and the largest numbers that fp16 has,
// 0.002 for heads of 256, otherwise far less.  With a larger scale, groups of 64 with nothing larger count as beyond fp16.
#define KV4_SMALL_SCALE 0.125f
#define KV4_SMALL 0x1p-14f

__host__ __device__ constexpr int kv4_record(int d) { return 9 * d; }
__host__ __device__ constexpr int kv4_values_at(int d) { return 4 * d; }
__host__ __device__ constexpr int kv4_key_params_at(int d) { return 8 * d; }
__host__ __device__ constexpr int kv4_value_params_at(int d) { return 8 * d + d / 2; }

// Byte (in the record) of the code of number i of token tok's key or value; bit 0 of i chooses the half.
__host__ __device__ constexpr int kv4_key_byte(int d, int tok, int i) {
  return tok * (d / 2) + (i % 64) / 16 * (d / 8) + i / 64 * 8 + (i % 16) / 2;
}
__host__ __device__ constexpr int kv4_value_byte(int d, int tok, int i) {
  return 4 * d + (i % 64) / 8 * (d / 2) + tok * (d / 16) + i / 64 * 4 + (i % 8) / 2;
}

// (s, m) as stored: s in the low half
__device__ __forceinline__ float kv4_scale(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float kv4_low(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }

// x - lo, at least zero.  Where a float does not hold it (numbers of far apart sizes) its last bit is one: it lies on the
// side of a border between codes, (c + 1/2) s of some thirteen bits, that the exact difference lies on.
__device__ __forceinline__ float kv4_above(float x, float lo) {
  const unsigned down = __float_as_uint(__fsub_rd(x, lo)), up = __float_as_uint(__fsub_ru(x, lo));
  return __uint_as_float(down | ((down ^ up) & 1u));
}

// The code of a number, whatever its size: on x / 4, which is exact, so that no difference of finite numbers
// overflows.  s has eight bits, so that a quotient off a border by the difference's last bit is not rounded onto it.
static __device__ __noinline__ unsigned kv4_any_code(float x, float lo, float s) {
  return s > 0.f ? (unsigned)fminf(rintf(kv4_above(x * 0.25f, lo * 0.25f) / (s * 0.25f)), 15.f) : 0u;
}

// The codes of a group's numbers, from its extremes (NaN if one of them is).  As a rule (`quick`) the quotient is a
// product with 1 / s put right by its remainder; only where s or the range leaves the ordinary floats is it
// computed as above.
struct Kv4Coder {
  float lo, s, inverse, half, below;
  unsigned pair;                           // (s, m) as stored
  bool finite, quick;
  __device__ __forceinline__ Kv4Coder(__nv_bfloat16 lowest, __nv_bfloat16 highest) {
    lo = __bfloat162float(lowest);
    const float hi = __bfloat162float(highest);
    finite = hi < INFINITY && lo > -INFINITY;               // (NaN: neither)
    const __nv_bfloat16 sb =
        finite ? __float2bfloat16_rn((hi * 0.25f - lo * 0.25f) / 3.75f) : __ushort_as_bfloat16(0x7fc0);
    const __nv_bfloat16 mb = finite ? __float2bfloat16_rn(lo) : sb;
    pair = (unsigned)__bfloat16_as_ushort(sb) | (unsigned)__bfloat16_as_ushort(mb) << 16;
    s = __bfloat162float(sb);
    quick = s >= 1e-30f && hi - lo < 3e38f;
    inverse = __fdividef(1.f, s), half = 0.5f * s, below = __uint_as_float(__float_as_uint(half) - 1u);
  }
  // quick: the product with 1 / s to the nearest, which is within one of it; the exact remainder says
  // whether it is the nearest, and of two equally near ones the even one
  __device__ __forceinline__ float quick_code(float x) const {
    const float y = kv4_above(x, lo), u = fmaf(y, inverse, 12582912.f), c = u - 12582912.f, left = fmaf(-c, s, y);
    const float limit = __float_as_uint(u) & 1u ? below : half;
    return fabsf(left) > limit ? c + copysignf(1.f, left) : c;
  }
};

// WORDS words at p (aligned as their number allows) by the widest reads.
template <int WORDS>
__device__ __forceinline__ void kv4_words(unsigned (&w)[WORDS], const unsigned char* p) {
  if constexpr (WORDS >= 4) {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const unsigned*>(p);
  }
}

// Whether some row at positions first .. last sees a key of [j0, j1] (window 0: no window).
__device__ __forceinline__ bool kv4_seen(int j0, int j1, int first, int last, int window, int keep) {
  if (j0 > last) return false;
  return window <= 0 || j0 < keep || j1 > first - window;
}
