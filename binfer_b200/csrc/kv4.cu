// Keys and values into pages held in 4 bits, and out of them (layout: kv4.cuh).
//
// Of 64 numbers x of a row: m = min x, s = bf16((max x - min x) / 15), c = (x - m) / s to the nearest
// whole number (ties to even), at most 15; s = 0 gives c = 0.  A group with a number that is not finite
// has s = m = NaN: all of it reads as NaN.  Everything is computed on x / 4, which is exact, so that no
// difference of finite numbers overflows; x - m and s are short enough that the float quotient falls on
// the side of a border that the exact one falls on.
#include "common.cuh"
#include "kv4.cuh"

#define KS_THREADS 256

// Sixteen lanes take a group, a lane four numbers; units are (token, key or value, kv head, group) in
// the order in which rows lie in memory.
template <int D, bool VEC>
__global__ void __launch_bounds__(KS_THREADS)
kv4_store_kernel(const __nv_bfloat16* __restrict__ k, long long k_stride,
                 const __nv_bfloat16* __restrict__ v, long long v_stride,
                 const int* __restrict__ slots, unsigned char* __restrict__ cache, int T, int nkv,
                 int page_size, long long num_slots, int* __restrict__ err) {
  constexpr int NG = D / KV4_GROUP;
  bf_pdl_trigger();
  bf_pdl_wait();
  const int lane = threadIdx.x & 31, l = lane & 15;
  const long long units = (long long)T * 2 * nkv * NG;
  const long long unit = ((long long)blockIdx.x * KS_THREADS + threadIdx.x) >> 4;
  const bool on = unit < units;
  const long long u = on ? unit : units - 1;                // (whole warps take part in the shuffles)
  const int g = (int)(u % NG), h = (int)(u / NG % nkv);
  const bool is_v = u / (NG * nkv) % 2;
  const long long t = u / ((long long)NG * nkv * 2);
  const __nv_bfloat16* src = (is_v ? v + t * v_stride : k + t * k_stride) + (size_t)h * D + g * 64 + l * 4;
  float x[4];
  if (VEC) {
    const uint2 raw = *reinterpret_cast<const uint2*>(src);
    x[0] = __uint_as_float(raw.x << 16), x[1] = __uint_as_float(raw.x & 0xffff0000u);
    x[2] = __uint_as_float(raw.y << 16), x[3] = __uint_as_float(raw.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(src[i]);
  }
  const int slot = slots[t];
  bool finite = true;
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    finite &= fabsf(x[i]) < INFINITY;
    x[i] *= 0.25f;
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const unsigned bad = ~__ballot_sync(0xffffffffu, finite) & (lane < 16 ? 0xffffu : 0xffff0000u);
  const __nv_bfloat16 sb = bad ? __ushort_as_bfloat16(0x7fc0) : __float2bfloat16_rn((hi - lo) / 3.75f);
  const __nv_bfloat16 mb = bad ? __ushort_as_bfloat16(0x7fc0) : __float2bfloat16_rn(lo * 4.f);
  const float s4 = __bfloat162float(sb) * 0.25f;
  unsigned code = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = s4 > 0.f ? fminf(rintf((x[i] - lo) / s4), 15.f) : 0.f;
    code |= (unsigned)c << (4 * i);
  }
  code |= __shfl_down_sync(0xffffffffu, code, 1) << 16;     // even lanes: eight codes
  if (!on || slot < 0) return;
  if ((long long)slot >= num_slots) {
    if (l == 0) atomicOr(err, BF_ERR_SLOT);
    return;
  }
  const int page = slot / page_size, off = slot - page * page_size, tok = off % KV4_EIGHTH;
  unsigned char* rec = cache + (((size_t)page * nkv + h) * (page_size / KV4_EIGHTH) + off / KV4_EIGHTH) *
                                   kv4_record(D);
  const int i0 = g * 64 + l * 4;
  if (!(l & 1))
    *reinterpret_cast<unsigned*>(rec + (is_v ? kv4_value_byte(D, tok, i0) : kv4_key_byte(D, tok, i0))) = code;
  if (l == 0)
    *reinterpret_cast<unsigned*>(rec + (is_v ? kv4_value_params_at(D) : kv4_key_params_at(D)) +
                                 (tok * NG + g) * 4) =
        (unsigned)__bfloat16_as_ushort(sb) | (unsigned)__bfloat16_as_ushort(mb) << 16;
}

BF_EXPORT int bf_kv4_store(const void* k, long long k_stride, const void* v, long long v_stride,
                           const int* slots, void* cache, int T, int nkv, int d, int page_size,
                           long long num_slots, int* err, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (d != 64 && d != 128 && d != 256) return (int)cudaErrorInvalidValue;
  const long long units = (long long)T * 2 * nkv * (d / KV4_GROUP);
  const long long blocks = (units * 16 + KS_THREADS - 1) / KS_THREADS;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const bool vec = k_stride % 4 == 0 && v_stride % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 7) == 0;
  auto run = [&](auto kern) {
    return bf_launch_pdl(kern, dim3((unsigned)blocks), dim3(KS_THREADS), 0, stream,
                         (const __nv_bfloat16*)k, k_stride, (const __nv_bfloat16*)v, v_stride, slots,
                         (unsigned char*)cache, T, nkv, page_size, num_slots, err);
  };
  if (d == 64) return vec ? run(kv4_store_kernel<64, true>) : run(kv4_store_kernel<64, false>);
  if (d == 128) return vec ? run(kv4_store_kernel<128, true>) : run(kv4_store_kernel<128, false>);
  return vec ? run(kv4_store_kernel<256, true>) : run(kv4_store_kernel<256, false>);
}

// ------------------------------------------------------------------------------- out of the pages
// A block takes 64 tokens of one portion's context and one kv head and writes them as a bfloat16 page
// [64][d] of keys and one of values; block 0 of each head writes page 0, which is zero.  Where a portion's
// pages begin is a sum over the portions before it.  What no row of the portion sees is zero (a page of
// nothing else is left out and its place in the table is page 0).
template <int D>
__global__ void __launch_bounds__(256)
kv4_load_kernel(const unsigned char* __restrict__ cache, const int* __restrict__ block_tables,
                int table_stride, int table_rows, int table_width,
                const int* __restrict__ items, int n_items,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                int* __restrict__ tables_out, int* __restrict__ items_out, int out_pages, int nkv,
                int page_size, int num_pages, int window, int keep, int* __restrict__ err) {
  constexpr int NG = D / KV4_GROUP, REC = kv4_record(D);
  bf_pdl_trigger();
  bf_pdl_wait();
  __shared__ int sh_item, sh_base;
  const int page = blockIdx.x, h = blockIdx.y;              // 0: the zero page; else page - 1 of the contexts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t out_page = ((size_t)page * nkv + h) * 64 * D;
  if (page == 0) {
    for (int i = threadIdx.x; i < 64 * D / 8; i += 256) {
      reinterpret_cast<uint4*>(k_out + out_page)[i] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(v_out + out_page)[i] = make_uint4(0, 0, 0, 0);
    }
    if (h == 0 && items_out)
      for (int i = threadIdx.x; i < n_items * 4; i += 256) items_out[i] = i % 4 ? items[i] : i / 4;
    return;
  }
  if (warp == 0) {
    int running = 0, item = -1, base = 0, total = 0;
    for (int i0 = 0; i0 < n_items; i0 += 32) {
      const int i = i0 + lane;
      const int n = i < n_items ? (max(items[4 * i + 2] + items[4 * i + 3], 0) + 63) / 64 : 0;
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
      }
      running += __shfl_sync(0xffffffffu, incl, 31);
    }
    total = running;
    if (lane == 0) {
      sh_item = item;
      sh_base = base;
      if (page == 1 && h == 0 && total > out_pages - 1) atomicOr(err, BF_ERR_SPLITS);
    }
  }
  __syncthreads();
  const int item = sh_item;
  __nv_bfloat16 *ko = k_out + out_page, *vo = v_out + out_page;
  if (item < 0) {                                           // behind the last context
    for (int i = threadIdx.x; i < 64 * D / 8; i += 256) {
      reinterpret_cast<uint4*>(ko)[i] = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(vo)[i] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int b = items[4 * item], first = items[4 * item + 3], last = first + items[4 * item + 2] - 1;
  const int j64 = (page - 1 - sh_base) * 64;
  const bool seen = kv4_seen(j64, j64 + 63, first, last, window, keep);
  if (h == 0 && threadIdx.x == 0) tables_out[(size_t)item * (out_pages - 1) + j64 / 64] = seen ? page : 0;
  if (!seen) return;
  // a warp takes a record: eight tokens
  const int j8 = j64 + warp * 8;
  bool have = kv4_seen(j8, j8 + 7, first, last, window, keep);
  int pid = 0;
  if (have) {
    const int at = j8 / page_size;
    pid = at < table_width && b >= 0 && b < table_rows ? block_tables[(size_t)b * table_stride + at] : -1;
    if (pid < 0 || pid >= num_pages) {
      if (lane == 0) atomicOr(err, BF_ERR_PAGE);
      have = false;
    }
  }
  const unsigned char* rec =
      cache + (((size_t)(have ? pid : 0) * nkv + h) * (page_size / 8) + j8 % page_size / 8) * REC;
  const int r = lane >> 2, q = lane & 3;
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
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // keys: lane (r, q) has part q of token r
  const bool on = have && kv4_seen(j8 + r, j8 + r, first, last, window, keep);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint2 w = have ? *reinterpret_cast<const uint2*>(rec + r * (D / 2) + q * (D / 8) + g * 8) : make_uint2(0, 0);
    const unsigned par = have ? *reinterpret_cast<const unsigned*>(rec + kv4_key_params_at(D) + (r * NG + g) * 4) : 0u;
    const float s = kv4_scale(par), m = kv4_low(par);
    uint4* dst = reinterpret_cast<uint4*>(ko + (warp * 8 + r) * D + g * 64 + q * 16);
    dst[0] = on ? eight(w.x, s, m) : zero;
    dst[1] = on ? eight(w.y, s, m) : zero;
  }
  // values: lane (r, q) has part r of tokens 2 q and 2 q + 1
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int tok = 2 * q + e;
    const bool von = have && kv4_seen(j8 + tok, j8 + tok, first, last, window, keep);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const unsigned w = have ? *reinterpret_cast<const unsigned*>(rec + 4 * D + r * (D / 2) + tok * (D / 16) + g * 4) : 0u;
      const unsigned par = have ? *reinterpret_cast<const unsigned*>(rec + kv4_value_params_at(D) + (tok * NG + g) * 4) : 0u;
      *reinterpret_cast<uint4*>(vo + (warp * 8 + tok) * D + g * 64 + r * 8) =
          von ? eight(w, kv4_scale(par), kv4_low(par)) : zero;
    }
  }
}

// tables_out [n_items][out_pages - 1] must be zeroed by the caller's launch before this one.
BF_EXPORT int bf_kv4_load(const void* cache, const int* block_tables, int table_stride, int table_rows,
                          int table_width, const int* items, int n_items, void* k_out, void* v_out, int* tables_out,
                          int* items_out, int out_pages, int nkv, int d, int page_size, int num_pages,
                          int window, int keep, int* err, cudaStream_t stream) {
  if (n_items <= 0 || out_pages <= 1) return 0;
  const cudaError_t e = cudaMemsetAsync(tables_out, 0, (size_t)n_items * (out_pages - 1) * 4, stream);
  if (e != cudaSuccess) return (int)e;
  auto run = [&](auto kern) {
    return bf_launch_pdl(kern, dim3(out_pages, nkv), dim3(256), 0, stream, (const unsigned char*)cache,
                         block_tables, table_stride, table_rows, table_width, items, n_items, (__nv_bfloat16*)k_out,
                         (__nv_bfloat16*)v_out, tables_out, items_out, out_pages, nkv, page_size,
                         num_pages, window, keep, err);
  };
  if (d == 64) return run(kv4_load_kernel<64>);
  if (d == 128) return run(kv4_load_kernel<128>);
  if (d == 256) return run(kv4_load_kernel<256>);
  return (int)cudaErrorInvalidValue;
}
