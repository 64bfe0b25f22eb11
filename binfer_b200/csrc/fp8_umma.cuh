// Device-side pieces that the products of 8-bit operands share.
#pragma once
#include <cuda.h>
#include <stdint.h>

#include "fp8.cuh"
#include "gate_act.cuh"
#include "tma_utils.cuh"
#include "umma_utils.cuh"

#define FP8_MAX_EXPERTS 512

namespace {

constexpr int FK = 128;   // K per stage: 128 codes = 128 bytes = one swizzle row = one group of scales

// c = float, a = b = e4m3, both K-major
__device__ __forceinline__ uint32_t fp8_idesc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// The lane that issues a converged warp's products and commits, chosen once: the instructions below take
// its predicate (electing for each anew is 20 cycles of the 350 that a group's six took).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r;
}
// (K = 32 per instruction: 32 bytes along the swizzled row)
__device__ __forceinline__ void umma_fp8(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint64_t* bar, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(elected)
      : "memory");
}
// A tile of a matrix into L2: nothing is read by this kernel, so what a kernel before it still writes there is
// not missed (L2 is where all SMs meet).
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y)
               : "memory");
}
// A look at a barrier that does not wait.
__device__ __forceinline__ bool mbar_look(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// A wait whose first look, `seen`, was taken earlier, under other work (a look takes 100 cycles).
__device__ __forceinline__ bool mbar_seen_or_wait_warp(bool seen, uint64_t* bar, uint32_t parity,
                                                       volatile int* abort) {
  if (__all_sync(0xffffffffu, seen)) return true;
  return mbar_wait_warp(bar, parity, abort);
}
// Loads of 8 or 16 columns that are not waited for; the wait for all of them; and (behind it) the
// registers, of which nothing was to be read before.
__device__ __forceinline__ void tmem_ask(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ask(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_got() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tmem_have(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile(""
                 : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                   "+r"(r[i + 6]), "+r"(r[i + 7]));
}
// (a0, a1) += (x0, x1) * (f0, f1)
__device__ __forceinline__ void fma2v(float& a0, float& a1, uint32_t x0, uint32_t x1, float f0, float f1) {
  asm("{\n\t.reg .b64 a, x, f;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 f, {%4, %5};\n\t"
      "fma.rn.f32x2 a, x, f, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(x0), "r"(x1), "f"(f0), "f"(f1));
}
// Barrier among `threads` threads under a number, which also ANDs a predicate.
__device__ __forceinline__ bool named_all(int id, int threads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 q, %3, 0;\n\t"
      "barrier.cta.red.and.pred p, %1, %2, q;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// ---- rows that belong to experts: expert e's are starts[e] .. starts[e + 1] - 1
// In shared memory: the rows of every expert and how many tiles of `tile` rows there are before it.
// Whatever `starts` holds, the rows lie inside the matrix.  Without experts (starts null) all rows are
// one expert's.
struct RowTables {
  int *first, *end, *before;      // [E], [E], [E + 1]
};
__device__ __forceinline__ RowTables row_tables_at(void* smem, int E) {
  int* p = reinterpret_cast<int*>(smem);
  return RowTables{p, p + E, p + 2 * E};
}
__host__ __device__ __forceinline__ int row_tables_bytes(int E) { return ((3 * E + 1) * 4 + 127) & ~127; }
// by the whole block; a __syncthreads() behind it
__device__ __forceinline__ void fill_row_tables(const RowTables& t, const int* starts, int E, int rows,
                                                int tile) {
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int a = 0, b = rows;
    if (starts) {
      a = min(max(starts[e], 0), rows);
      b = max(min(starts[e + 1], rows), a);
    }
    t.first[e] = a;
    t.end[e] = b;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + (int)threadIdx.x;
      int n = e < E ? (t.end[e] - t.first[e] + tile - 1) / tile : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int m = __shfl_up_sync(0xffffffffu, n, o);
        if ((int)threadIdx.x >= o) n += m;
      }
      if (e < E) t.before[e + 1] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (threadIdx.x == 0) t.before[0] = 0;
  }
}
// Unit u of before[E] * tiles_f: an expert's tiles lie together, row tiles fastest (CTAs side by side
// read the same weights).
struct RowTile {
  int expert, ft, row0, row_end;
};
__device__ __forceinline__ RowTile row_tile(const RowTables& t, int E, int tiles_f, int tile, int u) {
  int lo = 0, hi = E;                               // before[lo] tiles_f <= u < before[hi] tiles_f
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long long)t.before[mid] * tiles_f <= u) lo = mid; else hi = mid;
  }
  const int n = t.before[lo + 1] - t.before[lo], v = u - t.before[lo] * tiles_f;
  return RowTile{lo, v / n, t.first[lo] + v % n * tile, t.end[lo]};
}

// A [rows, K] matrix of codes (rows ld bytes apart) in boxes of box_rows x 128, 128-byte swizzle.
static inline int fp8_map(CUtensorMap* map, const void* base, long long rows, long long K, long long ld,
                          int box_rows) {
  BfEncodeTiledFn enc = bf_encode_tiled();
  if (!enc) return (int)cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)FK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
                         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// sixteen codes, of which `left` are there (the others zero), on a 16-byte boundary
__device__ __forceinline__ uint4 fp8_sixteen(const uint8_t* p, int left) {
  if (left >= 16) return *reinterpret_cast<const uint4*>(p);
  uint32_t r[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < left) r[j >> 2] |= (uint32_t)p[j] << (8 * (j & 3));
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// Whether the loop's sum of a result's groups g0 .. g1 - 1 is off because of a factor that is no float of full precision
// (fp8.cuh; one taken as zero does no harm where the row's numbers are zeros, as in a padded batch), and that sum by
// multiply-adds.  scale_x(g), scale_w(g): the groups' scales; x(g, k), w(g, k): where their codes k .. k + 15 lie (k a
// multiple of 16).  K: columns in all.  By one thread; slow, and rare.
template <typename SX, typename SW, typename X>
__device__ bool fp8_any_odd(int g0, int g1, int K, SX scale_x, SW scale_w, X x) {
  for (int g = g0; g < g1; ++g) {
    if (!fp8_odd(scale_x(g), scale_w(g))) continue;
    if (fp8_factor(scale_x(g), scale_w(g)).after > 1.f) return true;
    uint32_t any = 0u;
#pragma unroll 4
    for (int k = 0; k < FK; k += 16) {
      const uint4 c = fp8_sixteen(x(g, k), K - g * FK - k);
      any |= c.x | c.y | c.z | c.w;
    }
    if (any & 0x7f7f7f7fu) return true;
  }
  return false;
}
template <typename SX, typename SW, typename X, typename W>
__device__ float fp8_sum_anew(int g0, int g1, int K, SX scale_x, SW scale_w, X x, W w) {
  float acc = 0.f;
  for (int g = g0; g < g1; ++g) {
    const Fp8Factor f = fp8_factor(scale_x(g), scale_w(g));
    float sum = 0.f;
#pragma unroll 2
    for (int k = 0; k < FK; k += 16) {
      const uint4 a4 = fp8_sixteen(x(g, k), K - g * FK - k), b4 = fp8_sixteen(w(g, k), K - g * FK - k);
      const uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float u[4], v[4];
        fp8_values4(a[i], u);
        fp8_values4(b[i], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = fmaf(u[j], v[j], sum);
      }
    }
    acc = fmaf(sum * f.before, f.after, acc);
  }
  return acc;
}

__device__ __forceinline__ float fp8_gate(int act, float g, float u, const BfGateConst& k) {
  return act == BF_ACT_CLAMPED ? bf_gate_mul_fast<BF_ACT_CLAMPED>(g, u, k)
                               : bf_gate_mul_fast<BF_ACT_SILU>(g, u, k);
}

}  // namespace
