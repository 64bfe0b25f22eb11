// Keys and values into pages held in 4 bits, and out of them (layout: kv4.cuh).
//
// Of 64 numbers x of a row: m = min x, s = bf16((max x - min x) / 15), c = (x - m) / s to the nearest
// whole number (ties to even), at most 15; s = 0 gives c = 0.  A group with a number that is not finite
// has s = m = NaN: all of it reads as NaN.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"

#define KS_THREADS 256
#define KV4_VALUE_UP 16.f       // fp16 values: 2^-18 is the smallest with all its bits, 4,062 the largest

// z / n for small z, with ceil(2^32 / n) (n = 1: 0, which stands for 2^32)
__device__ __forceinline__ int ks_row(int z, unsigned inverse) {
  return inverse ? (int)__umulhi((unsigned)z, inverse) : z;
}

// Four lanes take a group, a lane the sixteen numbers of its part of a key; units are (token, key or value,
// kv head, group) in the order in which rows lie in memory.  The kernel is bound by its instructions, so
// minimum and maximum are taken two bfloat16 numbers at a time and quotients are products (Kv4Coder; bfloat16
// numbers make ties common).  2,048 tokens of 8 heads of 128: 5.5 us (10.8 MB, 1.6 at the rate of a copy); 13
// tokens 2.1, the launch and one round trip.
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
  const Kv4Coder coder(__hmin_nan(lo2.x, lo2.y), __hmax_nan(hi2.x, hi2.y));
  unsigned code[2] = {0u, 0u};
  if (coder.quick) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};                    // four codes each, as a whole number
#pragma unroll
    for (int j = 15; j >= 0; --j) {
      const float x = j & 1 ? __uint_as_float(raw[j >> 1] & 0xffff0000u) : __uint_as_float(raw[j >> 1] << 16);
      sum[j >> 2] = fmaf(16.f, sum[j >> 2], coder.quick_code(x));
    }
    code[0] = (unsigned)sum[0] | (unsigned)sum[1] << 16;
    code[1] = (unsigned)sum[2] | (unsigned)sum[3] << 16;
  } else if (coder.finite) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = j & 1 ? __uint_as_float(raw[j >> 1] & 0xffff0000u) : __uint_as_float(raw[j >> 1] << 16);
      code[j >> 3] |= kv4_any_code(x, coder.lo, coder.s) << (4 * (j & 7));
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
        coder.pair;
}

struct Kv4StoreCall {
  const void* k;
  long long k_stride;
  const void* v;
  long long v_stride;
  const int* slots;
  void* cache;
  int T, nkv, d, page_size;
  long long num_slots;
  int* err;
  cudaStream_t stream;
};
BF_EXPORT int bf_kv4_store(const Kv4StoreCall* call) {
  const auto& [k, k_stride, v, v_stride, slots, cache, T, nkv, d, page_size, num_slots, err, stream] =
               *call;
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
template <bool B>
struct KvBool {
  static constexpr bool value = B;
};

// A block takes 64 tokens of one portion's context and every gridDim.y-th kv head and writes them as bfloat16
// pages [64][d] of keys and of values, a warp a record of eight tokens; the blocks of page 0 write zeros.
// Where a portion's pages begin is a sum over the portions before it; one that names a request, places or token
// rows that are not there, or more places than a row of the table has, has none, and one that the pages left have no
// room for has zeros: its row of the table, which no block of its own can be sure to write, and its pages.  What no row of the portion sees is
// zero (a page of nothing else is left out and its place in the table is page 0).  The blocks of a portion
// write its row of the table together.  4,096 tokens of 8 heads of 128: 6.0 us (21.5 MB, 3.3 at the rate of a copy),
// 8,448 10.8 (6.8): a block's way to its page, and stores.  Several heads a block, one after the other, took longer
// (12.4 against 10.8), and a warp's eights in the order of the codes left half of each 32-byte sector to a second store.
//
// For attention on the tensor cores (HALF) keys and values are fp16, values KV4_VALUE_UP times: a number
// m + s c has up to twelve bits, of which bfloat16 keeps eight (the result's error was 0.0036 of its rms
// with both in bfloat16, 0.0027 with the values and probabilities; its own rounding to bfloat16 alone is
// 0.0017).  A byte a record then says whether it holds a key or value beyond fp16's range, a group of values
// so small that fp16 has less than half a step of 2^-11 for its largest, a group of keys that is (`small_key`,
// where the scale makes it matter), or a value that is not finite (a
// probability of zero times such a value is NaN: whole tiles would carry it into rows that do not see it);
// attention_kv4.cu computes what is concerned from the codes.
template <int D, bool HALF>
__global__ void __launch_bounds__(256)
kv4_load_kernel(const unsigned char* __restrict__ cache, const int* __restrict__ block_tables,
                int table_stride, int table_rows, int table_width, const int* __restrict__ items, int n_items,
                int T, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                int* __restrict__ tables_out, int out_width, int* __restrict__ items_out,
                unsigned char* __restrict__ special, int* __restrict__ beyond, int out_pages, int nkv, int page_size,
                int num_pages, int window, int keep, float small_key, int* __restrict__ err) {
  constexpr int NG = D / KV4_GROUP, REC = kv4_record(D);
  bf_pdl_trigger();
  bf_pdl_wait();
  const int page = blockIdx.x;                              // 0: the zero page; else page - 1 of the contexts
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // pages of a portion; negative: an error bit
  auto pages_of = [&](int b, int row0, int rows, int first) {
    const long long n = (long long)rows + first;
    if (rows <= 0 && n <= 0) return 0;
    if (rows < 0 || first < 0 || b < 0 || b >= table_rows || n > (long long)table_width * page_size || row0 < 0 ||
        row0 > T - rows)
      return -BF_ERR_PAGE;
    return n > out_width * 64LL ? -BF_ERR_SPLITS : (int)((n + 63) / 64);
  };
  // the portion of this page, by every warp for itself
  int item = -1, base = 0, b = 0, first = 0, n_rows = 0;
  for (int i0 = 0, running = 0; i0 < n_items; i0 += 32) {
    const int i = i0 + lane;
    int of[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i < n_items) of[k] = items[4 * i + k];
    const int found = pages_of(of[0], of[1], of[2], of[3]), n = max(found, 0);
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
      b = __shfl_sync(0xffffffffu, of[0], who);
      n_rows = __shfl_sync(0xffffffffu, of[2], who);
      first = __shfl_sync(0xffffffffu, of[3], who);
    }
    if (page == 0 && blockIdx.y == 0 && warp == 0 && i < n_items) {
      // a context that the pages or the table have no room for: none of its rows is attended
      const bool fits = found >= 0 && running + incl <= out_pages - 1;
      if (!fits) atomicOr(err, found < 0 ? -found : BF_ERR_SPLITS);
      if (items_out) {
        items_out[4 * i] = i, items_out[4 * i + 1] = of[1];
        items_out[4 * i + 2] = fits ? of[2] : 0, items_out[4 * i + 3] = of[3];
      }
    }
    running += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (page == 0 && blockIdx.y == 0) {
    if (HALF)
      for (int i = tid; i < n_items * nkv; i += 256) beyond[i] = 0;
    long long to = 0;                                       // portions without pages, or without room for all of them
    for (int i = 0; i < n_items; ++i) {
      const int n = pages_of(items[4 * i], items[4 * i + 1], items[4 * i + 2], items[4 * i + 3]);
      to += max(n, 0);
      if (n <= 0 || to > out_pages - 1)
        for (int w = tid; w < out_width; w += 256) tables_out[(size_t)i * out_width + w] = 0;
    }
  }
  if (item >= 0 && (long long)base + (n_rows + first - 1) / 64 + 1 > out_pages - 1) item = -1;
  if (page == 0 || item < 0) {                              // the zero page, and pages of no portion with room
    for (int h = blockIdx.y; h < nkv; h += gridDim.y) {
      const size_t at = ((size_t)page * nkv + h) * 64 * D;
      for (int i = tid; i < 64 * D / 8; i += 256) {
        reinterpret_cast<uint4*>(k_out + at)[i] = zero;
        reinterpret_cast<uint4*>(v_out + at)[i] = zero;
      }
    }
    return;
  }
  const int last = first + n_rows - 1;
  const int place = page - 1 - base, n_places = last / 64 + 1;
  if (blockIdx.y == 0) {                                    // this block's part of the portion's row
    const int w1 = place + 1 < n_places ? (int)((long long)out_width * (place + 1) / n_places) : out_width;
    for (int w = (int)((long long)out_width * place / n_places) + tid; w < w1; w += 256)
      tables_out[(size_t)item * out_width + w] =
          w < n_places && kv4_seen(w * 64, w * 64 + 63, first, last, window, keep) ? base + w + 1 : 0;
  }
  const int j64 = place * 64;
  if (!kv4_seen(j64, j64 + 63, first, last, window, keep)) return;
  const int j8 = j64 + warp * 8;                            // the warp's record: eight tokens
  bool have = kv4_seen(j8, j8 + 7, first, last, window, keep);
  int pid = 0;
  if (have) {
    const int at = j8 / page_size;
    pid = at < table_width ? block_tables[(size_t)b * table_stride + at] : -1;
    if (pid < 0 || pid >= num_pages) {
      if (lane == 0 && blockIdx.y == 0) atomicOr(err, BF_ERR_PAGE);
      have = false;
      pid = 0;
    }
  }
  auto eight = [](unsigned codes, float s, float m, auto half) {
    uint4 o;
    unsigned* w = reinterpret_cast<unsigned*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = fmaf(s, (float)(codes >> (8 * i) & 15), m), c = fmaf(s, (float)(codes >> (8 * i + 4) & 15), m);
      if constexpr (decltype(half)::value) {
        const __half2 p = __floats2half2_rn(a, c);
        w[i] = *reinterpret_cast<const unsigned*>(&p);
      } else {
        const __nv_bfloat162 p = __floats2bfloat162_rn(a, c);
        w[i] = *reinterpret_cast<const unsigned*>(&p);
      }
    }
    return o;
  };
  const int r = lane >> 2, q = lane & 3;
  const bool on = have && kv4_seen(j8 + r, j8 + r, first, last, window, keep);
  const bool v_on[2] = {have && kv4_seen(j8 + 2 * q, j8 + 2 * q, first, last, window, keep),
                        have && kv4_seen(j8 + 2 * q + 1, j8 + 2 * q + 1, first, last, window, keep)};
  constexpr int KW = D / 32;                                // words of a lane's keys, and of its values
  for (int h = blockIdx.y; h < nkv; h += gridDim.y) {
    const unsigned char* rec = cache + (((size_t)pid * nkv + h) * (page_size / 8) + j8 % page_size / 8) * REC;
    __nv_bfloat16* ko = k_out + (((size_t)page * nkv + h) * 64 + warp * 8) * D;
    __nv_bfloat16* vo = v_out + (((size_t)page * nkv + h) * 64 + warp * 8) * D;
    // keys: lane (r, q) has part q of token r; values: part r of tokens 2 q and 2 q + 1
    unsigned kw[KW], vw[KW], kp[NG], vp[2 * NG];
    kv4_words<KW>(kw, rec + r * (D / 2) + q * (D / 8));
    kv4_words<NG>(kp, rec + kv4_key_params_at(D) + r * NG * 4);
    kv4_words<KW>(vw, rec + kv4_values_at(D) + r * (D / 2) + q * (D / 8));
    kv4_words<2 * NG>(vp, rec + kv4_value_params_at(D) + q * NG * 8);
    bool other = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float s = kv4_scale(kp[g]), m = kv4_low(kp[g]);
      // a row's four lanes change eights, so that each store fills its 32-byte sectors
      uint4* dst = reinterpret_cast<uint4*>(ko + r * D + g * 64 + q * 8);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int from = (lane & ~3) | half * 2 | q >> 1;
        const unsigned w0 = __shfl_sync(0xffffffffu, kw[2 * g], from), w1 = __shfl_sync(0xffffffffu, kw[2 * g + 1], from);
        dst[half * 4] = on ? eight(q & 1 ? w1 : w0, s, m, KvBool<HALF>()) : zero;
      }
      if (HALF) {
        const float most = fmaxf(fabsf(m), fabsf(fmaf(15.f, s, m)));
        other |= on && (most > 65000.f || (most > 0.f && most < small_key));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float vs = kv4_scale(vp[e * NG + g]);
        const float up = HALF ? KV4_VALUE_UP : 1.f, vm = kv4_low(vp[e * NG + g]);
        *reinterpret_cast<uint4*>(vo + (2 * q + e) * D + g * 64 + r * 8) =
            v_on[e] ? eight(vw[e * NG + g], vs * up, vm * up, KvBool<HALF>()) : zero;
        if (HALF) {
          const float most = fmaxf(fabsf(vm), fabsf(fmaf(15.f, vs, vm)));
          other |= v_on[e] && (vs != vs || most > 65000.f / KV4_VALUE_UP || (most > 0.f && most < 0x1p-18f));
        }
      }
    }
    if (HALF) {
      other = __any_sync(0xffffffffu, other);
      if (lane == 0) special[((size_t)page * nkv + h) * 8 + warp] = other;
    }
  }
}

// special (8 bytes a page and head) and beyond (n_items x nkv), both or neither: keys and values in fp16, for scores
// times `scale`.
struct Kv4LoadCall {
  const void* cache;
  const int* block_tables;
  int table_stride, table_rows, table_width;
  const int* items;
  int n_items, T;
  void* k_out, *v_out;
  int* tables_out;
  int out_width;
  int* items_out;
  void* special;
  int* beyond;
  int out_pages, nkv, d, page_size, num_pages, window, keep, sms;
  float scale;
  int* err;
  cudaStream_t stream;
};
BF_EXPORT int bf_kv4_load(const Kv4LoadCall* call) {
  const auto& [cache, block_tables, table_stride, table_rows, table_width, items, n_items, T, k_out, v_out,
               tables_out, out_width, items_out, special, beyond, out_pages, nkv, d, page_size, num_pages,
               window, keep, sms, scale, err, stream] = *call;
  if (n_items <= 0 || out_pages <= 1) return 0;
  if ((special != nullptr) != (beyond != nullptr)) return (int)cudaErrorInvalidValue;
  // heads apart where pages alone would leave SMs without blocks
  int parts = 1;
  while (parts < nkv && (long long)out_pages * parts < 4LL * sms) parts *= 2;
  if (parts > nkv) parts = nkv;
  auto run = [&](auto kern) {
    return bf_launch_pdl(kern, dim3(out_pages, parts), dim3(256), 0, stream, (const unsigned char*)cache,
                         block_tables, table_stride, table_rows, table_width, items, n_items, T,
                         (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, tables_out, out_width, items_out,
                         (unsigned char*)special, beyond, out_pages, nkv, page_size, num_pages, window, keep,
                         scale > KV4_SMALL_SCALE ? KV4_SMALL : 0.f, err);
  };
  if (d == 64) return special ? run(kv4_load_kernel<64, true>) : run(kv4_load_kernel<64, false>);
  if (d == 128) return special ? run(kv4_load_kernel<128, true>) : run(kv4_load_kernel<128, false>);
  if (d == 256) return special ? run(kv4_load_kernel<256, true>) : run(kv4_load_kernel<256, false>);
  return (int)cudaErrorInvalidValue;
}
