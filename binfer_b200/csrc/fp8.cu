// Activations and weights into 8 bits and back (the format: fp8.cuh).
//
// All kernels pass over the data once, with the numbers of a group in registers between the search for
// the largest and the rounding.  2,048 x 12,288 bfloat16 into codes: 17.3 us (4.4 TB/s; eight or nine integer
// instructions a number), float32 23.6 (5.4 TB/s); back as floats: 24 us (5.2 TB/s); a weight of 12,288 x 4,096: 31 us
// (4.8 TB/s; float32 43, 5.8 TB/s), back as floats 47 (5.3 TB/s).
#include "fp8.cuh"

namespace {

constexpr int F8_THREADS = 256;

// How a grid walks the groups of a matrix, `places` of them in a block's hands: `across` groups of a row
// side by side (a power of two), places / across rows at once; blockIdx.x counts the former, blockIdx.y
// the latter.
struct Fp8Walk {
  int shift;                                     // log2(across)
  dim3 grid;
};
Fp8Walk fp8_walk(int places, long long rows, int groups, int num_sms, int mats) {
  Fp8Walk w;
  w.shift = 0;
  while ((1 << w.shift) < places && (1 << w.shift) < groups) ++w.shift;
  const int x = (groups + (1 << w.shift) - 1) >> w.shift;
  const int at_once = places >> w.shift;
  long long y = (rows + at_once - 1) / at_once;
  const long long most = (8LL * num_sms + (long long)x * mats - 1) / ((long long)x * mats);   // 8 blocks an SM
  if (y > most) y = most;
  if (y > 65535) y = 65535;
  w.grid = dim3((unsigned)x, (unsigned)y, (unsigned)mats);
  return w;
}

// the codes of Fp8Sixteen<., 64>, of which `n` are there
__device__ __forceinline__ void fp8_store16(uint8_t* dst, const uint4& c, int n) {
  if (n >= 72) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(c.x, c.y);            // (rows of codes lie on 16-byte boundaries)
    *reinterpret_cast<uint2*>(dst + 64) = make_uint2(c.z, c.w);
  } else {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int at = j < 8 ? j : 56 + j;
      if (at < n) dst[at] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
  }
}

// Eight lanes a group, sixteen numbers each.  scales [groups, lds]: the rows' scales of one group of
// columns lie together, as the products that read them want them.
constexpr int F8_ROW_PLACES = F8_THREADS / 8;
template <typename T, bool VEC>
__global__ void __launch_bounds__(F8_THREADS)
fp8_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, long long ldc,
                float* __restrict__ scales, long long lds, int rows, int K, int groups, int shift) {
  BF_TRACE_POINT(10 * BF_TR_FP8_ROWS);
  bf_pdl_trigger();
  const int sub = threadIdx.x & 7, place = threadIdx.x >> 3;
  const int g = (blockIdx.x << shift) + (place & ((1 << shift) - 1));
  const int at_once = F8_ROW_PLACES >> shift;
  const int step = (int)gridDim.y * at_once;
  const int k = g * BF_FP8_GROUP + sub * 8, n = g < groups ? K - k : 0;
  const long long t0 = (long long)blockIdx.y * at_once + (place >> shift);
  // (every lane of a block takes as many turns: the shuffles are the whole warp's)
  const int turns = (rows - (int)blockIdx.y * at_once + step - 1) / step;
  bf_pdl_wait();
  BF_TRACE_POINT(10 * BF_TR_FP8_ROWS + 1);
  for (int i = 0; i < turns; ++i) {
    const long long t = t0 + (long long)i * step;
    Fp8Sixteen<T, 64> v;
    const T* src = x + t * ldx + k;
    if (VEC && n >= 72 && t < rows) {
      v.template load<true>(src, n);
    } else {
      v.template load<false>(src, t < rows ? n : 0);
    }
    uint32_t m = v.largest();
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const Fp8Scale s = fp8_scale(m);
    if (t < rows && n > 0) fp8_store16(codes + t * ldc + k, v.codes(s), n);
    if (t < rows && g < groups && sub == 0) scales[g * lds + t] = s.s;
  }
  BF_TRACE_POINT(10 * BF_TR_FP8_ROWS + 2);
}

// A block a row: resid (+= delta), RMSNorm, rounding to bfloat16, into 8 bits; eight numbers a thread and
// trip, sixteen threads a group.  The sums have the order of the norm's own kernel: the codes are those of
// its output.  2,048 rows of 4,096 with an addition: 18.1 us (5.1 TB/s; the norm and fp8_rows one behind the other
// 22.1), 8 rows 2.6 (4.0): the way from the kernel ahead and two passes through a block's barrier.
template <int TRIPS>
__global__ void add_rmsnorm_fp8_kernel(float* __restrict__ resid, const __nv_bfloat16* __restrict__ delta,
                                       const float* __restrict__ w, uint8_t* __restrict__ codes, long long ldc,
                                       float* __restrict__ scales, long long lds, int H, float eps) {
  __shared__ float scratch[33];
  BF_TRACE_POINT(10 * BF_TR_FP8_NORM);
  bf_pdl_trigger();
  // (into L2 ahead of the wait, and no further: a kernel before this one may write the norm's weight)
#pragma unroll
  for (int k = 0; k < TRIPS; ++k) {
    const int c = (k * blockDim.x + threadIdx.x) * 8;
    if (c < H && threadIdx.x % 4 == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(w + c));
  }
  bf_pdl_wait();
  BF_TRACE_POINT(10 * BF_TR_FP8_NORM + 1);
  const int r = blockIdx.x;
  float* x = resid + (size_t)r * H;
  const __nv_bfloat16* d = delta ? delta + (size_t)r * H : nullptr;
  float v[TRIPS][8], f[TRIPS][8];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < TRIPS; ++k) {
    const int c = (k * blockDim.x + threadIdx.x) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    if (c < H) {
      const float4 wa = *reinterpret_cast<const float4*>(w + c);
      const float4 wb = *reinterpret_cast<const float4*>(w + c + 4);
      f[k][0] = wa.x; f[k][1] = wa.y; f[k][2] = wa.z; f[k][3] = wa.w;
      f[k][4] = wb.x; f[k][5] = wb.y; f[k][6] = wb.z; f[k][7] = wb.w;
      const float4 a = *reinterpret_cast<const float4*>(x + c);
      const float4 b = *reinterpret_cast<const float4*>(x + c + 4);
      v[k][0] = a.x; v[k][1] = a.y; v[k][2] = a.z; v[k][3] = a.w;
      v[k][4] = b.x; v[k][5] = b.y; v[k][6] = b.z; v[k][7] = b.w;
      if (d) {
        const uint4 q = *reinterpret_cast<const uint4*>(d + c);
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __bfloat1622float2(h[j]);
          v[k][2 * j] += f.x;
          v[k][2 * j + 1] += f.y;
        }
        *reinterpret_cast<float4*>(x + c) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        *reinterpret_cast<float4*>(x + c + 4) = make_float4(v[k][4], v[k][5], v[k][6], v[k][7]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v[k][j] * v[k][j];
    }
  }
  ss = block_sum(ss, scratch);
  const float inv = rsqrtf(ss / (float)H + eps);
#pragma unroll
  for (int k = 0; k < TRIPS; ++k) {
    const int c = (k * blockDim.x + threadIdx.x) * 8;
    uint32_t m = 0u;
    if (c < H) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[k][j] = __bfloat162float(__float2bfloat16_rn(v[k][j] * inv * f[k][j]));
        m = max(m, __float_as_uint(v[k][j]) & 0x7fffffffu);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const Fp8Scale s = fp8_scale(m);
    if (c < H) {
      uint32_t q[2], sg[2] = {0u, 0u};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sg[j >> 2] |= (__float_as_uint(v[k][j]) >> 31) << (8 * (j & 3) + 7);
        v[k][j] = fabsf(v[k][j]);
      }
      fp8_codes(v[k], sg, s, q);
      *reinterpret_cast<uint2*>(codes + r * ldc + c) = make_uint2(q[0], q[1]);
      if ((threadIdx.x & 15) == 0) scales[(long long)(c / BF_FP8_GROUP) * lds + r] = s.s;
    }
  }
  BF_TRACE_POINT(10 * BF_TR_FP8_NORM + 2);
}

// A warp a group, four numbers a lane: a warp's loads and stores are whole lines.  Eight rows a turn (8,192 x
// 12,288 to float32: 95.8 us, 102 with four).  Stores that leave L2 first would gain nothing but a rewrite of
// the same place, and cost the result's reader a tenth.
// blockIdx.z: the matrix, of mat_rows rows.  BLOCKS: a scale per 128 rows of it and group, [blocks, groups];
// else one per row and group, [groups, lds].
constexpr int F8_READ_PLACES = F8_THREADS / 32, F8_READ_TURN = 8;
template <typename T, bool BLOCKS>
__global__ void __launch_bounds__(F8_THREADS)
fp8_read_kernel(const uint8_t* __restrict__ codes, long long ldc, const float* __restrict__ scales,
                long long lds, T* __restrict__ out, long long ldo, int mat_rows, int K, int groups, int shift,
                bool vec) {
  bf_pdl_trigger();
  const int lane = threadIdx.x & 31, place = threadIdx.x >> 5;
  const int g = (blockIdx.x << shift) + (place & ((1 << shift) - 1)), r = place >> shift;
  const int at_once = F8_READ_PLACES >> shift;
  const long long step = (long long)gridDim.y * at_once;
  const int k = g * BF_FP8_GROUP + lane * 4, n = g < groups ? min(4, K - k) : 0;
  bf_pdl_wait();
  if (n <= 0) return;
  codes += (long long)blockIdx.z * mat_rows * ldc;
  out += (long long)blockIdx.z * mat_rows * ldo;
  if (BLOCKS) scales += (long long)blockIdx.z * ((mat_rows + BF_FP8_GROUP - 1) / BF_FP8_GROUP) * groups;
  for (long long t0 = (long long)blockIdx.y * at_once + r; t0 < mat_rows; t0 += F8_READ_TURN * step) {
    uint32_t c[F8_READ_TURN];
    float s[F8_READ_TURN];
#pragma unroll
    for (int i = 0; i < F8_READ_TURN; ++i) {
      const long long t = t0 + i * step;
      c[i] = 0u;
      s[i] = 0.f;
      if (t < mat_rows) {
        const uint8_t* src = codes + t * ldc + k;
        s[i] = BLOCKS ? scales[(t / BF_FP8_GROUP) * groups + g] : scales[g * lds + t];
        if (n == 4) {
          c[i] = *reinterpret_cast<const uint32_t*>(src);
        } else {
          for (int j = 0; j < n; ++j) c[i] |= (uint32_t)src[j] << (8 * j);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < F8_READ_TURN; ++i) {
      const long long t = t0 + i * step;
      if (t >= mat_rows) break;
      float v[4];
      fp8_values4(c[i], v);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= s[i];
      T* dst = out + t * ldo + k;
      if (vec && n == 4) {
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
          uint2 o;
          __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
          o2[0] = __floats2bfloat162_rn(v[0], v[1]);
          o2[1] = __floats2bfloat162_rn(v[2], v[3]);
          *reinterpret_cast<uint2*>(dst) = o;
        }
      } else {
        for (int j = 0; j < n; ++j) bf_st(dst + j, v[j]);
      }
    }
  }
}

// A block of 128 x 128 per CTA: 8 lanes a row, 32 rows at a time, four such passes held in registers.
// blockIdx: (group, block of rows, matrix).
template <typename T, bool VEC>
__global__ void __launch_bounds__(F8_THREADS)
fp8_blocks_kernel(const T* __restrict__ w, long long ldw, uint8_t* __restrict__ codes, long long ldc,
                  float* __restrict__ scales, int mat_rows, int K) {
  __shared__ uint32_t warp_max[F8_THREADS / 32];
  const int sub = threadIdx.x & 7, lead = threadIdx.x >> 3;
  const int g = blockIdx.x, r0 = blockIdx.y * BF_FP8_GROUP;
  const long long first = (long long)blockIdx.z * mat_rows;
  const int k = g * BF_FP8_GROUP + sub * 8, n = K - k;
  Fp8Sixteen<T, 64> v[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + i * 32 + lead, there = r < mat_rows ? n : 0;
    const T* src = w + (first + r) * ldw + k;
    if (VEC && there >= 72) {
      v[i].template load<true>(src, there);
    } else {
      v[i].template load<false>(src, there);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, v[i].largest());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < F8_THREADS / 32; ++i) m = max(m, warp_max[i]);
  const Fp8Scale s = fp8_scale(m);
  if (threadIdx.x == 0) scales[((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + g] = s.s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + i * 32 + lead;
    if (r < mat_rows && n > 0) fp8_store16(codes + (first + r) * ldc + k, v[i].codes(s), n);
  }
}

bool on_16(const void* p, long long ld, int size) {
  return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0;
}

}  // namespace

// x [rows, K] (float or bfloat16, rows ldx apart) -> codes [rows, ldc bytes], scales [ceil(K / 128), lds].
// codes: on a 16-byte boundary, ldc a multiple of 16.
struct Fp8RowsCall {
  const void* x;
  long long ldx;
  void* codes;
  long long ldc;
  float* scales;
  long long lds;
  int dtype, rows, K, num_sms;
  cudaStream_t stream;
};
BF_EXPORT int bf_fp8_rows(const Fp8RowsCall* call) {
  const auto& [x, ldx, codes, ldc, scales, lds, dtype, rows, K, num_sms, stream] = *call;
  if (rows <= 0 || K <= 0) return 0;
  if (!on_16(codes, ldc, 1)) return (int)cudaErrorInvalidValue;
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const Fp8Walk walk = fp8_walk(F8_ROW_PLACES, rows, groups, num_sms, 1);
  uint8_t* c = (uint8_t*)codes;
  auto go = [&](auto kern, auto* src) {
    return bf_launch_pdl(kern, walk.grid, dim3(F8_THREADS), 0, call->stream, src, call->ldx, c, call->ldc,
                         call->scales, call->lds, call->rows, call->K, groups, walk.shift);
  };
  if (dtype == BF_DTYPE_F32) {
    const float* f = (const float*)x;
    return on_16(x, ldx, 4) ? go(fp8_rows_kernel<float, true>, f) : go(fp8_rows_kernel<float, false>, f);
  }
  const __nv_bfloat16* h = (const __nv_bfloat16*)x;
  return on_16(x, ldx, 2) ? go(fp8_rows_kernel<__nv_bfloat16, true>, h)
                          : go(fp8_rows_kernel<__nv_bfloat16, false>, h);
}

// `mats` matrices of mat_rows x K one behind the other in w (rows ldw apart) -> codes the same way (rows
// ldc bytes apart), scales [mats, ceil(mat_rows / 128), ceil(K / 128)].
struct Fp8BlocksCall {
  const void* w;
  long long ldw;
  void* codes;
  long long ldc;
  float* scales;
  int dtype, mats, mat_rows, K;
  cudaStream_t stream;
};
BF_EXPORT int bf_fp8_blocks(const Fp8BlocksCall* call) {
  const auto& [w, ldw, codes, ldc, scales, dtype, mats, mat_rows, K, stream] = *call;
  if (mats <= 0 || mat_rows <= 0 || K <= 0) return 0;
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const int blocks = (mat_rows + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  if (!on_16(codes, ldc, 1) || mats > 65535 || blocks > 65535) return (int)cudaErrorInvalidValue;
  uint8_t* c = (uint8_t*)codes;
  // (launched the ordinary way: what a model is loaded with gains nothing by an early start)
  auto go = [&](auto kern, auto* src) {
    kern<<<dim3(groups, blocks, call->mats), F8_THREADS, 0, call->stream>>>(
        src, call->ldw, c, call->ldc, call->scales, call->mat_rows, call->K);
    return bf_launch_status();
  };
  if (dtype == BF_DTYPE_F32) {
    const float* f = (const float*)w;
    return on_16(w, ldw, 4) ? go(fp8_blocks_kernel<float, true>, f) : go(fp8_blocks_kernel<float, false>, f);
  }
  const __nv_bfloat16* h = (const __nv_bfloat16*)w;
  return on_16(w, ldw, 2) ? go(fp8_blocks_kernel<__nv_bfloat16, true>, h)
                          : go(fp8_blocks_kernel<__nv_bfloat16, false>, h);
}

// What codes and scales stand for, into out (float or bfloat16, rows ldo apart): `mats` matrices of
// mat_rows x K one behind the other.  blocks: scales as bf_fp8_blocks leaves them, else as bf_fp8_rows.
struct Fp8ReadCall {
  const void* codes;
  long long ldc;
  const float* scales;
  long long lds;
  void* out;
  long long ldo;
  int dtype, blocks, mats, mat_rows, K, num_sms;
  cudaStream_t stream;
};
BF_EXPORT int bf_fp8_read(const Fp8ReadCall* call) {
  const auto& [codes, ldc, scales, lds, out, ldo, dtype, blocks, mats, mat_rows, K, num_sms, stream] = *call;
  if (mats <= 0 || mat_rows <= 0 || K <= 0) return 0;
  if (!on_16(codes, ldc, 1) || mats > 65535 || (!blocks && mats != 1)) return (int)cudaErrorInvalidValue;
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const Fp8Walk walk =
      fp8_walk(F8_READ_PLACES, (mat_rows + F8_READ_TURN - 1LL) / F8_READ_TURN, groups, num_sms, mats);
  auto go = [&](auto kern, auto* dst) {
    return bf_launch_pdl(kern, walk.grid, dim3(F8_THREADS), 0, call->stream, (const uint8_t*)call->codes,
                         call->ldc, call->scales, call->lds, dst, call->ldo, call->mat_rows, call->K, groups,
                         walk.shift, on_16(call->out, call->ldo, (int)sizeof(*dst)));
  };
  if (dtype == BF_DTYPE_F32)
    return blocks ? go(fp8_read_kernel<float, true>, (float*)out) : go(fp8_read_kernel<float, false>, (float*)out);
  return blocks ? go(fp8_read_kernel<__nv_bfloat16, true>, (__nv_bfloat16*)out)
                : go(fp8_read_kernel<__nv_bfloat16, false>, (__nv_bfloat16*)out);
}

// resid [rows, H] += delta (bfloat16, or null); its RMSNorm times w, rounded to bfloat16, as codes [rows, ldc
// bytes] and scales [ceil(H / 128), lds].  H: a multiple of 8, at most 8,192; everything on 16-byte boundaries.
struct AddRmsnormFp8Call {
  float* resid;
  const void* delta;
  const float* w;
  void* codes;
  long long ldc;
  float* scales;
  long long lds;
  int rows, H;
  float eps;
  cudaStream_t stream;
};
BF_EXPORT int bf_add_rmsnorm_fp8(const AddRmsnormFp8Call* call) {
  const AddRmsnormFp8Call& c = *call;
  if (c.rows <= 0) return 0;
  if (c.H % 8 || c.H <= 0 || c.H > 8 * 256 * 4 || c.ldc % 16 ||
      (((uintptr_t)c.resid | (uintptr_t)c.delta | (uintptr_t)c.w | (uintptr_t)c.codes) & 15))
    return (int)cudaErrorInvalidValue;
  const int threads = c.H >= 2048 ? 256 : 128, trips = (c.H / 8 + threads - 1) / threads;
  auto go = [&](auto kern) {
    return bf_launch_pdl(kern, dim3(c.rows), dim3(threads), 0, c.stream, c.resid, (const __nv_bfloat16*)c.delta,
                         c.w, (uint8_t*)c.codes, c.ldc, c.scales, c.lds, c.H, c.eps);
  };
  if (trips <= 1) return go(add_rmsnorm_fp8_kernel<1>);
  if (trips == 2) return go(add_rmsnorm_fp8_kernel<2>);
  return go(add_rmsnorm_fp8_kernel<4>);
}

extern "C" int bf_gemm_fp8_few(const void*, long long, const float*, long long, const void*, long long,
                               const float*, const int*, const float*, void*, long long, int, int, int, int,
                               int, int, int, float, float, float, int, int, int, int, int*, cudaStream_t);
extern "C" int bf_gemm_fp8_pair(const void*, long long, const float*, long long, const void*, long long,
                                const float*, const int*, const float*, void*, long long, int, int, int, int,
                                int, int, int, float, float, float, int, int, int*, cudaStream_t);

// How a product runs: the most rows of a tile of gemm_fp8_few.cu, or -1 for gemm_fp8_pair.cu.
// Without experts: tiles of 32 rows while there is one for every SM at most, or two with few groups (157
// rows, 6,144 x 4,096: 17.2 us against 22.3 with tiles of 64 and 18.0 on pairs; 4,096 x 12,288: 36.9 / 38.0 /
// 32.1); then 64 if those hold all rows (64 rows, 24,576 x 4,096 gated: 33.1 / 27.0 / 42.3); up to 96 rows 32
// again (35.2 / 48.9 / 42.8); then pairs (157 rows of the same: 57.1 / 50.0 / 43.7).
// With experts by the rows that one has on average (64 experts, 2,048 x 2,048 gated, 8 to 128 rows each: 52 /
// 52 / 53 us with tiles of 16 / 32 / 64 and 80 on pairs, 58 / 57 / 56 / 83, 99 / 72 / 67 / 88, 188 / 131 / 108 / 96).
// The rows' shares lie on the device and are not known here: where few experts have all rows, theirs come in more
// and smaller tiles than would be fastest.
static int fp8_tile(int rows, int features, int K, bool gated, int experts, int num_sms) {
  const int each = (rows + experts - 1) / experts;
  if (each <= 16) return 16;
  if (experts > 1) return each <= 24 ? 32 : each <= 112 ? 64 : -1;
  if (each <= 32) return 32;
  const long long tiles = (rows + 31LL) / 32 * ((features + (gated ? 63 : 127)) / (gated ? 64 : 128));
  if (tiles <= num_sms || (tiles <= 2 * num_sms && K <= 48 * BF_FP8_GROUP)) return 32;
  if (each <= 64) return 64;
  return each <= 96 && tiles <= 4 * num_sms ? 32 : -1;
}
// CTAs that share a tile of 128 weight rows: as many (a power of two: clusters of other sizes leave SMs
// of a GPC empty) as are resident together, two to an SM, each with two groups at least.
static int fp8_split(int rows, int features, int K, bool gated, int nb, int num_sms) {
  const long long tiles = (long long)((rows + nb - 1) / nb) * ((features + (gated ? 63 : 127)) / (gated ? 64 : 128));
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  int c = 1;
  while (c < 8 && tiles * 2 * c <= 2 * num_sms && groups >= 4 * c) c *= 2;
  return c;
}

// Pairs that share a tile of 256 x 256, each with four groups at least: two while those are resident together
// (157 rows, 4,096 x 12,288: 47.2 -> 32.6 us; 512 rows: 50.6 -> 37.1), four for the fewest tiles (64 rows, 1,024
// x 4,096: 18.7 / 15.4 / 13.6; with 16 tiles, whose clusters of eight CTAs run in two turns, 19.5 / 16.4 / 27.4).
static int fp8_pair_split(int rows, int features, int K, bool gated, int num_sms) {
  const long long tiles = (rows + 255LL) / 256 * ((features + (gated ? 127 : 255)) / (gated ? 128 : 256));
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  if (tiles * 16 <= num_sms && groups >= 16) return 4;
  return tiles * 4 <= num_sms * 9LL / 10 && groups >= 8 ? 2 : 1;
}

struct Fp8ProductCall {
  const void* x;               // bfloat16 [rows, K], or null: codes and scales hold the rows
  long long ldx;
  void* codes;                 // scratch for the rows' codes and scales
  long long ldc;
  float* scales;
  long long lds;
  const void* w;
  long long ldw;
  const float* sw;
  const int* starts;
  const float* row_w;
  void* out;
  long long ldo;
  int out_dtype, rows, features, K, experts, gated, act;
  float limit, slope, up_offset;
  int tile, split, num_sms;    // tile, split: 0 chosen here
  int* err;
  cudaStream_t stream;
};
// The rows into 8 bits, and their product with a held weight (bf_gemm_fp8_few's arguments).  Without scratch
// (codes null): as one kernel, or -1 and nothing done where that does not take the sizes.
BF_EXPORT int bf_fp8_product(const Fp8ProductCall* call) {
  const Fp8ProductCall& c = *call;
  if (c.rows <= 0 || c.features <= 0) return 0;
  const int tile = c.tile ? c.tile : fp8_tile(c.rows, c.features, c.K, c.gated != 0, c.experts, c.num_sms);
  const int split = c.starts ? 1
                    : c.split ? c.split
                    : tile < 0 ? fp8_pair_split(c.rows, c.features, c.K, c.gated != 0, c.num_sms)
                               : fp8_split(c.rows, c.features, c.K, c.gated != 0, tile, c.num_sms);
  if (c.x && !c.codes) {
    // asked for without scratch: the rows stay in the CTAs that read them, where they fit
    if (tile != 16 || c.starts) return -1;
    return bf_gemm_fp8_few(c.x, c.ldx, nullptr, 0, c.w, c.ldw, c.sw, c.starts, c.row_w, c.out, c.ldo, c.out_dtype,
                           c.rows, c.features, c.K, c.experts, c.gated, c.act, c.limit, c.slope, c.up_offset,
                           tile, split, 1, c.num_sms, c.err, c.stream);
  }
  const Fp8RowsCall rows = {c.x, c.ldx, c.codes, c.ldc, c.scales, c.lds, BF_DTYPE_BF16, c.rows, c.K, c.num_sms,
                            c.stream};
  const int e = c.x ? bf_fp8_rows(&rows) : 0;
  if (e) return e;
  if (tile < 0)
    return bf_gemm_fp8_pair(c.codes, c.ldc, c.scales, c.lds, c.w, c.ldw, c.sw, c.starts, c.row_w, c.out, c.ldo,
                            c.out_dtype, c.rows, c.features, c.K, c.experts, c.gated, c.act, c.limit, c.slope,
                            c.up_offset, split, c.num_sms, c.err, c.stream);
  return bf_gemm_fp8_few(c.codes, c.ldc, c.scales, c.lds, c.w, c.ldw, c.sw, c.starts, c.row_w, c.out, c.ldo,
                         c.out_dtype, c.rows, c.features, c.K, c.experts, c.gated, c.act, c.limit, c.slope,
                         c.up_offset, tile, split, 0, c.num_sms, c.err, c.stream);
}

BF_TRACE_READER(bf_trace_read_fp8)
