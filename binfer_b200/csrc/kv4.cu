// Keys and values into pages held in 4 bits, and out of them (layout: kv4.cuh).
//
// Of 64 numbers x of a row: m = min x, s = bf16((max x - min x) / 15), c = (x - m) / s to the nearest
// whole number (ties to even), at most 15; s = 0 gives c = 0.  A group with a number that is not finite
// has s = m = NaN: all of it reads as NaN.
#include "common.cuh"
#include "kv4.cuh"

#define KS_THREADS 256

// z / n for small z, with ceil(2^32 / n) (n = 1: 0, which stands for 2^32)
__device__ __forceinline__ int ks_row(int z, unsigned inverse) {
  return inverse ? (int)__umulhi((unsigned)z, inverse) : z;
}

// The code of a number, whatever its size: on x / 4, which is exact, so that no difference of finite numbers
// overflows.  x - m and s are short enough that the float quotient falls on the side of a border that
// the exact one falls on.
__device__ __noinline__ unsigned ks_code(float x, float lo, float s) {
  return s > 0.f ? (unsigned)fminf(rintf((x * 0.25f - lo * 0.25f) / (s * 0.25f)), 15.f) : 0u;
}

// Four lanes take a group, a lane the sixteen numbers of its part of a key; units are (token, key or value,
// kv head, group) in the order in which rows lie in memory.  The kernel is bound by its instructions, so
// minimum and maximum are taken two bfloat16 numbers at a time and the quotient is a product with 1 / s put
// right by its remainder (bfloat16 numbers make ties common); only where s or the range leaves the ordinary
// floats is it computed as above.
template <int D, bool VEC>
__global__ void __launch_bounds__(KS_THREADS)
kv4_store_kernel(const __nv_bfloat16* __restrict__ k, long long k_stride,
                 const __nv_bfloat16* __restrict__ v, long long v_stride,
                 const int* __restrict__ slots, unsigned char* __restrict__ cache, int units, int nkv,
                 unsigned row_inverse, int page_shift, long long num_slots, int* __restrict__ err) {
  constexpr int NG = D / KV4_GROUP, TEAMS = KS_THREADS / 4;
  bf_pdl_trigger();
  bf_pdl_wait();
  const int l = threadIdx.x & 3, team = threadIdx.x >> 2;
  const int per_row = NG * nkv, first = blockIdx.x * TEAMS, first_row = first / per_row;
  const bool on = first + team < units;                     // (whole warps take part in the shuffles)
  const int z = on ? first - first_row * per_row + team : 0;
  const int over = ks_row(z, row_inverse), i = z - over * per_row, row = first_row + over, t = row >> 1;
  const bool is_v = row & 1;
  const __nv_bfloat16* src = (is_v ? v + t * v_stride : k + t * k_stride) + i * 64 + l * 16;
  unsigned raw[8];
  if (VEC) {
    const uint4 a = reinterpret_cast<const uint4*>(src)[0], b = reinterpret_cast<const uint4*>(src)[1];
    raw[0] = a.x, raw[1] = a.y, raw[2] = a.z, raw[3] = a.w, raw[4] = b.x, raw[5] = b.y, raw[6] = b.z, raw[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      raw[j] = (unsigned)__bfloat16_as_ushort(src[2 * j]) | (unsigned)__bfloat16_as_ushort(src[2 * j + 1]) << 16;
  }
  const int slot = on ? slots[t] : -1;
  auto two = [&](int j) { return *reinterpret_cast<const __nv_bfloat162*>(&raw[j]); };
  __nv_bfloat162 lo2 = two(0), hi2 = two(0);
#pragma unroll
  for (int j = 1; j < 8; ++j) lo2 = __hmin2_nan(lo2, two(j)), hi2 = __hmax2_nan(hi2, two(j));
#pragma unroll
  for (int o = 2; o; o >>= 1) {
    lo2 = __hmin2_nan(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
    hi2 = __hmax2_nan(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
  }
  if (slot < 0) return;
  if ((long long)slot >= num_slots) {
    if (l == 0) atomicOr(err, BF_ERR_SLOT);
    return;
  }
  const float lo = __bfloat162float(__hmin_nan(lo2.x, lo2.y)), hi = __bfloat162float(__hmax_nan(hi2.x, hi2.y));
  const bool finite = hi < INFINITY && lo > -INFINITY;      // (NaN: neither)
  const __nv_bfloat16 sb = finite ? __float2bfloat16_rn((hi * 0.25f - lo * 0.25f) / 3.75f) : __ushort_as_bfloat16(0x7fc0);
  const __nv_bfloat16 mb = finite ? __float2bfloat16_rn(lo) : sb;
  const float s = __bfloat162float(sb);
  unsigned code[2] = {0u, 0u};
  if (s >= 1e-30f && hi - lo < 3e38f) {
    // c: the product with 1 / s to the nearest, which is within one of it; the exact remainder says
    // whether it is the nearest, and of two equally near ones the even one
    const float inverse = __fdividef(1.f, s), half = 0.5f * s, below = __uint_as_float(__float_as_uint(half) - 1u);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};                    // four codes each, as a whole number
#pragma unroll
    for (int j = 15; j >= 0; --j) {
      const float x = j & 1 ? __uint_as_float(raw[j >> 1] & 0xffff0000u) : __uint_as_float(raw[j >> 1] << 16);
      const float y = x - lo, u = fmaf(y, inverse, 12582912.f), c = u - 12582912.f, left = fmaf(-c, s, y);
      const float limit = __float_as_uint(u) & 1u ? below : half;
      sum[j >> 2] = fmaf(16.f, sum[j >> 2], fabsf(left) > limit ? c + copysignf(1.f, left) : c);
    }
    code[0] = (unsigned)sum[0] | (unsigned)sum[1] << 16;
    code[1] = (unsigned)sum[2] | (unsigned)sum[3] << 16;
  } else if (finite) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = j & 1 ? __uint_as_float(raw[j >> 1] & 0xffff0000u) : __uint_as_float(raw[j >> 1] << 16);
      code[j >> 3] |= ks_code(x, lo, s) << (4 * (j & 7));
    }
  }
  const int h = i / NG, g = i % NG, tok = slot % KV4_EIGHTH;
  unsigned char* rec = cache + ((((size_t)(slot >> page_shift) * nkv + h) << (page_shift - 3)) +
                                ((slot & ((1 << page_shift) - 1)) >> 3)) * kv4_record(D);
  if (is_v) {                                               // parts 2 l and 2 l + 1
    unsigned char* dst = rec + 4 * D + l * D + tok * (D / 16) + g * 4;
    *reinterpret_cast<unsigned*>(dst) = code[0];
    *reinterpret_cast<unsigned*>(dst + D / 2) = code[1];
  } else {
    *reinterpret_cast<uint2*>(rec + tok * (D / 2) + l * (D / 8) + g * 8) = make_uint2(code[0], code[1]);
  }
  if (l == 0)
    *reinterpret_cast<unsigned*>(rec + (is_v ? kv4_value_params_at(D) : kv4_key_params_at(D)) + (tok * NG + g) * 4) =
        (unsigned)__bfloat16_as_ushort(sb) | (unsigned)__bfloat16_as_ushort(mb) << 16;
}

BF_EXPORT int bf_kv4_store(const void* k, long long k_stride, const void* v, long long v_stride,
                           const int* slots, void* cache, int T, int nkv, int d, int page_size,
                           long long num_slots, int* err, cudaStream_t stream) {
  if (T <= 0) return 0;
  if ((d != 64 && d != 128 && d != 256) || page_size < 8 || (page_size & (page_size - 1)))
    return (int)cudaErrorInvalidValue;
  const int per_row = nkv * (d / KV4_GROUP);
  const long long units = (long long)T * 2 * per_row;
  if (units > 0x3fffffffLL || per_row > 1 << 14) return (int)cudaErrorInvalidValue;
  int page_shift = 3;
  while (1 << page_shift < page_size) ++page_shift;
  const unsigned blocks = (unsigned)((units * 4 + KS_THREADS - 1) / KS_THREADS);
  // (exact for the z < per_row + 64 that come up)
  const unsigned row_inverse = per_row > 1 ? (unsigned)((0x100000000ULL + per_row - 1) / per_row) : 0u;
  const bool vec = k_stride % 8 == 0 && v_stride % 8 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  auto run = [&](auto kern) {
    return bf_launch_pdl(kern, dim3(blocks), dim3(KS_THREADS), 0, stream, (const __nv_bfloat16*)k, k_stride,
                         (const __nv_bfloat16*)v, v_stride, slots, (unsigned char*)cache, (int)units, nkv,
                         row_inverse, page_shift, num_slots, err);
  };
  if (d == 64) return vec ? run(kv4_store_kernel<64, true>) : run(kv4_store_kernel<64, false>);
  if (d == 128) return vec ? run(kv4_store_kernel<128, true>) : run(kv4_store_kernel<128, false>);
  return vec ? run(kv4_store_kernel<256, true>) : run(kv4_store_kernel<256, false>);
}

// ------------------------------------------------------------------------------- out of the pages
// A block takes 64 tokens of one portion's context and every gridDim.y-th kv head and writes them as bfloat16
// pages [64][d] of keys and of values, a warp a record of eight tokens; the blocks of page 0 write zeros.
// Where a portion's pages begin is a sum over the portions before it.  What no row of the portion sees is
// zero (a page of nothing else is left out and its place in the table is page 0).  The blocks of a portion
// write its row of the table together.
template <int D>
__global__ void __launch_bounds__(256)
kv4_load_kernel(const unsigned char* __restrict__ cache, const int* __restrict__ block_tables,
                int table_stride, int table_rows, int table_width, const int* __restrict__ items, int n_items,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                int* __restrict__ tables_out, int out_width, int* __restrict__ items_out,
                unsigned char* __restrict__ not_finite, int out_pages, int nkv, int page_size, int num_pages, int window, int keep, int* __restrict__ err) {
  constexpr int NG = D / KV4_GROUP, REC = kv4_record(D);
  bf_pdl_trigger();
  bf_pdl_wait();
  __shared__ int sh_item, sh_base, sh_of[4];
  const int page = blockIdx.x;                              // 0: the zero page; else page - 1 of the contexts
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (warp == 0) {
    int running = 0, item = -1, base = 0;
    for (int i0 = 0; i0 < n_items; i0 += 32) {
      const int i = i0 + lane;
      int of[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i < n_items) of[k] = items[4 * i + k];
      const int n = (max(of[2] + of[3], 0) + 63) / 64;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned mine = __ballot_sync(0xffffffffu, page - 1 >= running + incl - n && page - 1 < running + incl);
      if (mine) {
        const int who = __ffs(mine) - 1;
        item = i0 + who;
        base = running + __shfl_sync(0xffffffffu, incl - n, who);
        if (lane == who) {
#pragma unroll
          for (int k = 0; k < 4; ++k) sh_of[k] = of[k];
        }
      }
      if (page == 0 && blockIdx.y == 0 && i < n_items) {
        // a context that the pages or the table have no room for: none of its rows is attended
        const bool fits = running + incl <= out_pages - 1 && n <= out_width;
        if (!fits) atomicOr(err, BF_ERR_SPLITS);
        if (items_out) {
          items_out[4 * i] = i, items_out[4 * i + 1] = of[1];
          items_out[4 * i + 2] = fits ? of[2] : 0, items_out[4 * i + 3] = of[3];
        }
      }
      running += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      sh_item = item;
      sh_base = base;
    }
  }
  __syncthreads();
  const int item = sh_item;
  if (page == 0 && blockIdx.y == 0) {
    for (int i = 0; i < n_items; ++i)                       // (portions without a page of their own)
      if (items[4 * i + 2] + items[4 * i + 3] <= 0)
        for (int w = tid; w < out_width; w += 256) tables_out[(size_t)i * out_width + w] = 0;
  }
  if (page == 0 || item < 0) {                              // the zero page, and pages behind the last context
    for (int h = blockIdx.y; h < nkv; h += gridDim.y) {
      const size_t at = ((size_t)page * nkv + h) * 64 * D;
      for (int i = tid; i < 64 * D / 8; i += 256) {
        reinterpret_cast<uint4*>(k_out + at)[i] = zero;
        reinterpret_cast<uint4*>(v_out + at)[i] = zero;
      }
    }
    return;
  }
  const int b = sh_of[0], first = sh_of[3], last = first + sh_of[2] - 1;
  const int place = page - 1 - sh_base, n_places = last / 64 + 1;
  if (blockIdx.y == 0) {                                    // this block's part of the portion's row
    const int w1 = place + 1 < n_places ? (int)((long long)out_width * (place + 1) / n_places) : out_width;
    for (int w = (int)((long long)out_width * place / n_places) + tid; w < w1; w += 256)
      tables_out[(size_t)item * out_width + w] =
          w < n_places && sh_base + w + 1 < out_pages && kv4_seen(w * 64, w * 64 + 63, first, last, window, keep)
              ? sh_base + w + 1 : 0;
  }
  const int j64 = place * 64;
  if (!kv4_seen(j64, j64 + 63, first, last, window, keep)) return;
  const int j8 = j64 + warp * 8;                            // the warp's record: eight tokens
  bool have = kv4_seen(j8, j8 + 7, first, last, window, keep);
  int pid = 0;
  if (have) {
    const int at = j8 / page_size;
    pid = at < table_width && b >= 0 && b < table_rows ? block_tables[(size_t)b * table_stride + at] : -1;
    if (pid < 0 || pid >= num_pages) {
      if (lane == 0 && blockIdx.y == 0) atomicOr(err, BF_ERR_PAGE);
      have = false;
      pid = 0;
    }
  }
  auto eight = [](unsigned codes, float s, float m) {
    uint4 o;
    unsigned* w = reinterpret_cast<unsigned*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = fmaf(s, (float)(codes >> (8 * i) & 15), m), c = fmaf(s, (float)(codes >> (8 * i + 4) & 15), m);
      __nv_bfloat162 p = __floats2bfloat162_rn(a, c);
      w[i] = *reinterpret_cast<unsigned*>(&p);
    }
    return o;
  };
  const int r = lane >> 2, q = lane & 3;
  const bool on = have && kv4_seen(j8 + r, j8 + r, first, last, window, keep);
  const bool v_on[2] = {have && kv4_seen(j8 + 2 * q, j8 + 2 * q, first, last, window, keep),
                        have && kv4_seen(j8 + 2 * q + 1, j8 + 2 * q + 1, first, last, window, keep)};
  for (int h = blockIdx.y; h < nkv; h += gridDim.y) {
    const unsigned char* rec =
        cache + (((size_t)pid * nkv + h) * (page_size / 8) + j8 % page_size / 8) * REC;
    __nv_bfloat16* ko = k_out + (((size_t)page * nkv + h) * 64 + warp * 8) * D;
    __nv_bfloat16* vo = v_out + (((size_t)page * nkv + h) * 64 + warp * 8) * D;
    uint2 kw[NG];
    unsigned vw[2][NG], kp[NG], vp[2][NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {                          // keys: lane (r, q) has part q of token r
      kw[g] = *reinterpret_cast<const uint2*>(rec + r * (D / 2) + q * (D / 8) + g * 8);
      kp[g] = *reinterpret_cast<const unsigned*>(rec + kv4_key_params_at(D) + (r * NG + g) * 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {                         // values: part r of tokens 2 q and 2 q + 1
        vw[e][g] = *reinterpret_cast<const unsigned*>(rec + 4 * D + r * (D / 2) + (2 * q + e) * (D / 16) + g * 4);
        vp[e][g] = *reinterpret_cast<const unsigned*>(rec + kv4_value_params_at(D) + ((2 * q + e) * NG + g) * 4);
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float s = kv4_scale(kp[g]), m = kv4_low(kp[g]);
      uint4* dst = reinterpret_cast<uint4*>(ko + r * D + g * 64 + q * 16);
      dst[0] = on ? eight(kw[g].x, s, m) : zero;
      dst[1] = on ? eight(kw[g].y, s, m) : zero;
      unsigned nan = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float vs = kv4_scale(vp[e][g]);
        bool write = v_on[e];
        if (not_finite && write && vs != vs) {              // noted in its place, see kv4_poison_kernel
          nan |= 1u << (2 * q + e);
          write = false;
        }
        *reinterpret_cast<uint4*>(vo + (2 * q + e) * D + g * 64 + r * 8) =
            write ? eight(vw[e][g], vs, kv4_low(vp[e][g])) : zero;
      }
      if (not_finite) {
        nan = __reduce_or_sync(0xffffffffu, nan);
        if (lane == 0) not_finite[((((size_t)page * nkv + h) * NG) + g) * 8 + warp] = (unsigned char)nan;
      }
    }
  }
}

BF_EXPORT int bf_kv4_load(const void* cache, const int* block_tables, int table_stride, int table_rows,
                          int table_width, const int* items, int n_items, void* k_out, void* v_out,
                          int* tables_out, int out_width, int* items_out, void* not_finite, int out_pages,
                          int nkv, int d, int page_size, int num_pages, int window, int keep, int sms, int* err,
                          cudaStream_t stream) {
  if (n_items <= 0 || out_pages <= 1) return 0;
  // heads apart where pages alone would leave SMs without blocks
  int parts = 1;
  while (parts < nkv && (long long)out_pages * parts < 4LL * sms) parts *= 2;
  if (parts > nkv) parts = nkv;
  auto run = [&](auto kern) {
    return bf_launch_pdl(kern, dim3(out_pages, parts), dim3(256), 0, stream, (const unsigned char*)cache,
                         block_tables, table_stride, table_rows, table_width, items, n_items,
                         (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, tables_out, out_width, items_out,
                         (unsigned char*)not_finite, out_pages, nkv, page_size, num_pages, window, keep, err);
  };
  if (d == 64) return run(kv4_load_kernel<64>);
  if (d == 128) return run(kv4_load_kernel<128>);
  if (d == 256) return run(kv4_load_kernel<256>);
  return (int)cudaErrorInvalidValue;
}

// A probability of zero times a value that is not finite is NaN, so a product over whole tiles would
// carry a token's values into rows that do not see it.  Where the caller attends over the loaded pages, such
// groups of values are therefore zero in them and noted (a bit a token, [page][head][group][64]), and this
// kernel writes NaN where a row sees one.  As a rule none is noted and a block only reads a few words.
template <int NG>
__global__ void __launch_bounds__(256)
kv4_poison_kernel(const unsigned long long* __restrict__ not_finite, const int* __restrict__ items,
                  const int* __restrict__ tables, int width, __nv_bfloat16* __restrict__ out,
                  long long out_stride, int T, int nkv, int group, int window, int keep) {
  const int h = blockIdx.x, item = blockIdx.y;
  bf_pdl_trigger();
  bf_pdl_wait();
  const int row0 = items[4 * item + 1], rows = items[4 * item + 2], first = items[4 * item + 3];
  const int places = min((first + rows + 63) / 64, width);
  const int* table = tables + (size_t)item * width;
  bool any = false;
  for (int w = threadIdx.x; w < places; w += 256) {
    const int page = table[w];
    if (page <= 0) continue;
    for (int g = 0; g < NG; ++g) any |= not_finite[((size_t)page * nkv + h) * NG + g] != 0;
  }
  if (!__syncthreads_or(any)) return;
  for (int i = threadIdx.x; i < rows * NG; i += 256) {
    const int row = i / NG, g = i - row * NG, p = first + row;
    bool sees = false;
    for (int w = 0; w < places && w * 64 <= p && !sees; ++w) {
      const int page = table[w];
      unsigned long long bits = page > 0 ? not_finite[((size_t)page * nkv + h) * NG + g] : 0ULL;
      for (; bits && !sees; bits &= bits - 1) {
        const int j = w * 64 + __ffsll(bits) - 1;
        sees = j <= p && (window <= 0 || j > p - window || j < keep);
      }
    }
    if (!sees || row0 + row >= T) continue;
    for (int c = 0; c < group; ++c)
      for (int e = 0; e < 64; ++e)
        out[(long long)(row0 + row) * out_stride + ((size_t)(h * group + c) * NG + g) * 64 + e] =
            __ushort_as_bfloat16(0x7fc0);
  }
}

BF_EXPORT int bf_kv4_poison(const void* not_finite, const int* items, int n_items, const int* tables, int width,
                            void* out, long long out_stride, int T, int nh, int nkv, int d, int window, int keep,
                            cudaStream_t stream) {
  if (n_items <= 0) return 0;
  auto run = [&](auto kern) {
    return bf_launch_pdl(kern, dim3(nkv, n_items), dim3(256), 0, stream, (const unsigned long long*)not_finite,
                         items, tables, width, (__nv_bfloat16*)out, out_stride, T, nkv, nh / nkv, window, keep);
  };
  if (d == 64) return run(kv4_poison_kernel<1>);
  if (d == 128) return run(kv4_poison_kernel<2>);
  if (d == 256) return run(kv4_poison_kernel<4>);
  return (int)cudaErrorInvalidValue;
}
