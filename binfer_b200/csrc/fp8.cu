// Activations and weights into 8 bits and back (the format: fp8.cuh).
//
// All four kernels pass over the data once, with the numbers of a group in registers between the
// search for the largest and the rounding; what bounds them is memory.
#include "fp8.cuh"

namespace {

constexpr int ROWS_THREADS = 256;

// 16 lanes hold a group of 128 numbers of a row, eight each; groups of a row side by side.
// scales [groups, lds]: the rows' scales of one group of columns lie together, as the products that
// read them want them.
template <typename T, bool VEC>
__global__ void __launch_bounds__(ROWS_THREADS)
fp8_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, long long ldc,
                float* __restrict__ scales, long long lds, int rows, int K, int groups) {
  bf_pdl_trigger();
  bf_pdl_wait();
  const int sub = threadIdx.x & 15;
  const long long total = (long long)rows * groups;
  const long long step = (long long)gridDim.x * (ROWS_THREADS / 16);
  const long long first = (long long)blockIdx.x * (ROWS_THREADS / 16) + threadIdx.x / 16;
  // (both halves of a warp take as many turns: the shuffles below are the whole warp's)
  for (long long i = first; i - (first & 1) < total; i += step) {
    const bool there = i < total;
    const int t = there ? (int)(i / groups) : 0, g = there ? (int)(i - (long long)t * groups) : 0;
    const int k = g * BF_FP8_GROUP + sub * 8, n = there ? min(8, K - k) : 0;
    float v[8];
    const T* src = x + (long long)t * ldx + k;
    if (VEC && n == 8) {
      fp8_load8<true>(src, 8, v);
    } else {
      fp8_load8<false>(src, n, v);
    }
    uint32_t m = fp8_largest8(v);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float s = fp8_scale(m), inv = __fdiv_rn(1.f, s);
    if (n > 0) {
      const uint2 c = make_uint2(fp8_codes4(v, s, inv), fp8_codes4(v + 4, s, inv));
      uint8_t* dst = codes + (long long)t * ldc + k;         // (ldc: a multiple of 16)
      if (n == 8) {
        *reinterpret_cast<uint2*>(dst) = c;
      } else {
        for (int j = 0; j < n; ++j) dst[j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
      }
    }
    if (there && sub == 0) scales[(long long)g * lds + t] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(ROWS_THREADS)
fp8_read_kernel(const uint8_t* __restrict__ codes, long long ldc, const float* __restrict__ scales,
                long long lds, T* __restrict__ out, long long ldo, long long rows, int K, int groups,
                int block_rows, int mat_rows, int mat_blocks, bool vec) {
  bf_pdl_trigger();
  bf_pdl_wait();
  const int sub = threadIdx.x & 15;
  const long long total = rows * groups;
  for (long long i = (long long)blockIdx.x * (ROWS_THREADS / 16) + threadIdx.x / 16; i < total;
       i += (long long)gridDim.x * (ROWS_THREADS / 16)) {
    const long long t = i / groups;
    const int g = (int)(i - t * groups);
    const int k = g * BF_FP8_GROUP + sub * 8, n = min(8, K - k);
    if (n <= 0) continue;
    // (rows: a scale per row and group, groups first; blocks: one per 128 rows of a matrix and group)
    const float s = block_rows == 1
                        ? scales[(long long)g * lds + t]
                        : scales[((t / mat_rows) * mat_blocks + t % mat_rows / block_rows) * groups + g];
    const uint8_t* src = codes + t * ldc + k;
    uint2 c;
    if (n == 8) {
      c = *reinterpret_cast<const uint2*>(src);
    } else {
      c = make_uint2(0u, 0u);
      for (int j = 0; j < n; ++j) (j < 4 ? c.x : c.y) |= (uint32_t)src[j] << (8 * (j & 3));
    }
    float v[8];
    fp8_values4(c.x, v);
    fp8_values4(c.y, v + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= s;
    T* dst = out + t * ldo + k;
    if (vec && n == 8) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        uint4 o;
        __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
        for (int j = 0; j < 4; ++j) o2[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<uint4*>(dst) = o;
      }
    } else {
      for (int j = 0; j < n; ++j) bf_st(dst + j, v[j]);
    }
  }
}

// A block of 128 x 128 per CTA: 16 lanes a row, 16 rows at a time, eight such passes held in registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
fp8_blocks_kernel(const T* __restrict__ w, long long ldw, uint8_t* __restrict__ codes, long long ldc,
                  float* __restrict__ scales, int mat_rows, int mat_blocks, int K, int groups) {
  __shared__ uint32_t warp_max[8];
  const int sub = threadIdx.x & 15, lead = threadIdx.x >> 4;
  const int g = blockIdx.x % groups;
  const long long b = blockIdx.x / groups;                     // block row over all matrices
  const long long mat = b / mat_blocks;
  const int r0 = (int)(b - mat * mat_blocks) * BF_FP8_GROUP;
  const int k = g * BF_FP8_GROUP + sub * 8, n = min(8, K - k);
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i * 16 + lead, nn = r < mat_rows ? n : 0;
    const T* src = w + (mat * mat_rows + r) * ldw + k;
    if (VEC && nn == 8) {
      fp8_load8<true>(src, 8, v[i]);
    } else {
      fp8_load8<false>(src, nn, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, fp8_largest8(v[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, warp_max[i]);
  const float s = fp8_scale(m), inv = __fdiv_rn(1.f, s);
  if (threadIdx.x == 0) scales[b * groups + g] = s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i * 16 + lead;
    if (r >= mat_rows || n <= 0) continue;
    const uint2 c = make_uint2(fp8_codes4(v[i], s, inv), fp8_codes4(v[i] + 4, s, inv));
    uint8_t* dst = codes + (mat * mat_rows + r) * ldc + k;
    if (n == 8) {
      *reinterpret_cast<uint2*>(dst) = c;
    } else {
      for (int j = 0; j < n; ++j) dst[j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
    }
  }
}

int blocks_for(long long items, int num_sms) {
  const long long blocks = (items + ROWS_THREADS / 16 - 1) / (ROWS_THREADS / 16);
  const long long most = 8LL * num_sms;                       // 8 blocks of 256 threads an SM
  return (int)(blocks < most ? blocks : most);
}

bool on_16(const void* p, long long ld, int size) {
  return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0;
}

}  // namespace

// x [rows, K] (float or bfloat16, rows ldx apart) -> codes [rows, ldc bytes], scales [ceil(K / 128), lds].
// codes: on a 16-byte boundary, ldc a multiple of 16.
BF_EXPORT int bf_fp8_rows(const void* x, long long ldx, int dtype, void* codes, long long ldc,
                          float* scales, long long lds, int rows, int K, int num_sms,
                          cudaStream_t stream) {
  if (rows <= 0 || K <= 0) return 0;
  if (!on_16(codes, ldc, 1)) return (int)cudaErrorInvalidValue;
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const dim3 grid(blocks_for((long long)rows * groups, num_sms));
  const int size = dtype == BF_DTYPE_F32 ? 4 : 2;
  const bool vec = on_16(x, ldx, size);
  uint8_t* c = (uint8_t*)codes;
#define BF_GO(T, V)                                                                              \
  return bf_launch_pdl(fp8_rows_kernel<T, V>, grid, dim3(ROWS_THREADS), 0, stream, (const T*)x, ldx, c, \
                       ldc, scales, lds, rows, K, groups)
  if (dtype == BF_DTYPE_F32) {
    if (vec) BF_GO(float, true);
    BF_GO(float, false);
  }
  if (vec) BF_GO(__nv_bfloat16, true);
  BF_GO(__nv_bfloat16, false);
#undef BF_GO
}

// `mats` matrices of mat_rows x K one behind the other in w (rows ldw apart) -> codes the same way (rows
// ldc bytes apart), scales [mats, ceil(mat_rows / 128), ceil(K / 128)].
BF_EXPORT int bf_fp8_blocks(const void* w, long long ldw, int dtype, void* codes, long long ldc,
                            float* scales, int mats, int mat_rows, int K, cudaStream_t stream) {
  if (mats <= 0 || mat_rows <= 0 || K <= 0) return 0;
  if (!on_16(codes, ldc, 1)) return (int)cudaErrorInvalidValue;
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const int blocks = (mat_rows + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const long long total = (long long)mats * blocks * groups;
  if (total > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const dim3 grid((unsigned)total);
  const int size = dtype == BF_DTYPE_F32 ? 4 : 2;
  const bool vec = on_16(w, ldw, size);
  uint8_t* c = (uint8_t*)codes;
  // (launched the ordinary way, and no kernel behind it may begin before it has ended: the products
  // ask for weights ahead of their wait for the kernels before them)
#define BF_GO(T, V)                                                                               \
  {                                                                                               \
    fp8_blocks_kernel<T, V><<<grid, 256, 0, stream>>>((const T*)w, ldw, c, ldc, scales, mat_rows, \
                                                      blocks, K, groups);                         \
    return bf_launch_status();                                                                    \
  }
  if (dtype == BF_DTYPE_F32) {
    if (vec) BF_GO(float, true);
    BF_GO(float, false);
  }
  if (vec) BF_GO(__nv_bfloat16, true);
  BF_GO(__nv_bfloat16, false);
#undef BF_GO
}

// What codes and scales stand for, into out (float or bfloat16, rows ldo apart).  block_rows 1: scales
// [ceil(K / 128), lds]; 128: `rows` rows of matrices of mat_rows each, scales as bf_fp8_blocks leaves them.
BF_EXPORT int bf_fp8_read(const void* codes, long long ldc, const float* scales, long long lds, void* out,
                          long long ldo, int dtype, long long rows, int K, int block_rows, int mat_rows,
                          int num_sms, cudaStream_t stream) {
  if (rows <= 0 || K <= 0) return 0;
  if (!on_16(codes, ldc, 1) || (block_rows != 1 && block_rows != BF_FP8_GROUP) || mat_rows <= 0)
    return (int)cudaErrorInvalidValue;
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const int mat_blocks = (mat_rows + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  const dim3 grid(blocks_for(rows * groups, num_sms));
  if (dtype == BF_DTYPE_F32)
    return bf_launch_pdl(fp8_read_kernel<float>, grid, dim3(ROWS_THREADS), 0, stream,
                         (const uint8_t*)codes, ldc, scales, lds, (float*)out, ldo, rows, K, groups,
                         block_rows, mat_rows, mat_blocks, on_16(out, ldo, 4));
  return bf_launch_pdl(fp8_read_kernel<__nv_bfloat16>, grid, dim3(ROWS_THREADS), 0, stream,
                       (const uint8_t*)codes, ldc, scales, lds, (__nv_bfloat16*)out, ldo, rows, K, groups,
                       block_rows, mat_rows, mat_blocks, on_16(out, ldo, 2));
}

extern "C" int bf_gemm_fp8_few(const void*, long long, const float*, long long, const void*, long long,
                               const float*, const int*, const float*, void*, long long, int, int, int, int,
                               int, int, int, float, float, float, int, int, int, int*, cudaStream_t);
extern "C" int bf_gemm_fp8_pair(const void*, long long, const float*, long long, const void*, long long,
                                const float*, const int*, const float*, void*, long long, int, int, int, int,
                                int, int, int, float, float, float, int, int*, cudaStream_t);

// How a product runs: the most rows of a tile of gemm_fp8_few.cu, or -1 for gemm_fp8_pair.cu.
static int fp8_tile(int rows, int experts) {
  const int each = (rows + experts - 1) / experts;
  if (each > 256) return -1;
  int nb = 16;
  while (nb < each) nb *= 2;
  return nb;
}
// CTAs that share a tile of 128 weight rows: as many as the SMs have room for, each with two groups
static int fp8_split(int rows, int features, int K, bool gated, int nb, int num_sms) {
  const int tiles = ((rows + nb - 1) / nb) * ((features + (gated ? 63 : 127)) / (gated ? 64 : 128));
  const int groups = (K + BF_FP8_GROUP - 1) / BF_FP8_GROUP;
  int c = 1;
  while (c < 8 && tiles * (c + 1) <= num_sms && groups >= 2 * (c + 1)) ++c;
  return nb <= 64 ? c : 1;
}

struct Fp8ProductCall {
  const void* x;               // bfloat16 [rows, K]
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
// The rows into 8 bits, and their product with a held weight (bf_gemm_fp8_few's arguments).
BF_EXPORT int bf_fp8_product(const Fp8ProductCall* call) {
  const Fp8ProductCall& c = *call;
  if (c.rows <= 0 || c.features <= 0) return 0;
  const int e = bf_fp8_rows(c.x, c.ldx, BF_DTYPE_BF16, c.codes, c.ldc, c.scales, c.lds, c.rows, c.K, c.num_sms,
                            c.stream);
  if (e) return e;
  const int tile = c.tile ? c.tile : fp8_tile(c.rows, c.experts);
  if (tile < 0)
    return bf_gemm_fp8_pair(c.codes, c.ldc, c.scales, c.lds, c.w, c.ldw, c.sw, c.starts, c.row_w, c.out, c.ldo,
                            c.out_dtype, c.rows, c.features, c.K, c.experts, c.gated, c.act, c.limit, c.slope,
                            c.up_offset, c.num_sms, c.err, c.stream);
  const int split = c.starts ? 1
                    : c.split ? c.split
                              : fp8_split(c.rows, c.features, c.K, c.gated != 0, tile, c.num_sms);
  return bf_gemm_fp8_few(c.codes, c.ldc, c.scales, c.lds, c.w, c.ldw, c.sw, c.starts, c.row_w, c.out, c.ldo,
                         c.out_dtype, c.rows, c.features, c.K, c.experts, c.gated, c.act, c.limit, c.slope,
                         c.up_offset, tile, split, c.num_sms, c.err, c.stream);
}
