// Products with weights in 8 bits for many rows: the sums of gemm_fp8_few.cu on pairs of SMs.
//
// Tiles of 256 activation rows x 256 weight rows, a cluster of two CTAs each (tcgen05.mma.cta_group::2.
// kind::f8f6f4): a CTA holds 128 rows of the activations in its lanes of tensor memory and fetches half
// of the weight rows.  Here the activations are the product's rows, so that a thread has one row's
// scale and the weight's scale is one number a group: one multiplication a group of 128 instead of one
// factor per column.  The sums of a group (256 columns) go into one of two buffers of tensor memory;
// sixteen warps per CTA, four to a quarter of the lanes, add them times the factor into 64 registers each
// while the products fill the other buffer.
//
//   warp 0       TMA: 128 activation rows and 128 weight rows x 128 bytes per stage
//   warp 1       (leader) the products; TMEM allocation
//   warps 2, 3   look for products of two scales that are no floats of full precision
//   warps 4-19   the sums into registers; the result, turned in shared memory so that a warp writes
//                64 bytes a row (these four warpgroups take 112 registers a thread, which the first
//                leaves them: 128 x 32 + 512 x 112 of the launch's 640 x 96; with 104 the products of 2,048
//                rows and 24,576 x 4,096 gated took 210 us, with 112 201)
//
// What bounds it: the sums' warps.  A group's products take 512 cycles, its 32 packed multiply-adds a warp 278 for
// the four warps of a scheduler, but a warp executes 126 instructions a group in a chain of waits (2,048 rows,
// 24,576 x 4,096 gated, 205 us without the rows' codes, 2.0 PFLOP/s; parts left out to time the rest, of 201 us then:
// without fetching operands 6 us less, without the results 26, with an eighth of the multiply-adds 50; products and
// signals alone 110).  When it runs on, the clock too (1.67 GHz at 900 W).  Eight warps with 128 sums each took 236 us.
//
// SPLIT: few tiles leave SMs idle, and `split` pairs share one, a cluster of twice as many CTAs: each adds up
// its part of the groups, the parts meet in the shared memory that the ring had, a pair owning a slice of
// the columns, and are added to that pair's own in the pairs' order.
//
// Gated: a CTA's half of the weight rows are 64 gate rows and the 64 up rows of the same outputs, so a
// thread holds both.  With experts a tile's rows are one expert's.
//
// Every wait is bounded; no load uses multicast.
#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"
#include "fp8_umma.cuh"
#include "pair_utils.cuh"

namespace {

constexpr int PF_THREADS = 640;             // five warpgroups of 96 registers a thread at launch
constexpr int PF_SUMS = 16;                 // warps that add up the sums
constexpr int PF_TILE = 256;
constexpr int PF_HALF = 128 * FK;             // a CTA's rows of either operand
constexpr int PF_STAGE = 2 * PF_HALF;
constexpr int PF_STAGES = 5;
constexpr int PF_BARS = 512;
constexpr int PF_TURN = 32 * 64;              // a warp's rows on their way out: 32 x 64 bytes

// (128 bytes: of a longer one the compiler makes a copy, which cost 8,088 rows of a mixture 4 of 43 us)
struct PairParams {
  int rows, features, K, groups;
  int experts, tiles_f, w_blocks;
  int split;                            // SPLIT: 2 or 4
  const uint8_t *x, *w;                 // what the tensor maps show ...
  uint32_t ldx16, ldw16;                // ... whose rows are so many times 16 bytes apart
  const int* starts;
  const float* sx;
  long long lds;
  const float* sw;
  const float* row_w;
  long long ldo;
  int act;
  BfGateConst gk;
  int* err;
};
static_assert(sizeof(PairParams) <= 128, "see above");

__device__ __forceinline__ void pair_umma_fp8(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc,
                                              uint32_t idesc, uint32_t accumulate, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
// arrives on the barrier at this offset in both CTAs of the pair (`both`: their bits)
__device__ __forceinline__ void pair_commit_by(uint64_t* bar, uint32_t both, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;\n\t}" ::"r"(smem_u32(bar)),
      "h"((uint16_t)both), "r"(elected)
      : "memory");
}

// An arrival on a barrier of the cluster that orders no memory: what it tells of are reads of tensor
// memory, which tcgen05.wait::ld and tcgen05.fence have ended.  (With the default, a release at the
// cluster's scope, the warps stood at a memory barrier for most of a group's time: 2,048 x 4,096 against
// 8,192 rows gated took 196 us.)
__device__ __forceinline__ void pair_arrive_relaxed(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr)
               : "memory");
}

// 32 rows of a warp, 64 bytes each (a lane has a row, `v` its sixteen-byte pieces), to out: row r of the
// warp goes to dst + r * ldo, as far as there are rows and columns.
template <typename OutT>
__device__ __forceinline__ void turn_and_store(uint8_t* buf, const uint4 (&v)[4], OutT* dst, long long ldo,
                                               int n_rows, int n_cols, bool vec, int lane) {
  constexpr int PER = 16 / (int)sizeof(OutT);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = v[q];
  __syncwarp();
  const int q = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    const uint4 x = *reinterpret_cast<const uint4*>(buf + r * 64 + ((q ^ ((r >> 1) & 3)) << 4));
    if (r < n_rows && q * PER < n_cols) {
      OutT* d = dst + (long long)r * ldo + q * PER;
      if (vec && q * PER + PER <= n_cols) {
        *reinterpret_cast<uint4*>(d) = x;
      } else {
        const OutT* e = reinterpret_cast<const OutT*>(&x);
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (q * PER + j < n_cols) d[j] = e[j];
      }
    }
  }
  __syncwarp();
}

template <typename OutT, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(PF_THREADS, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                OutT* __restrict__ out, const PairParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  bf_pdl_trigger();
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(base);       // waited on in the leader only
  uint64_t* empty = full + PF_STAGES;
  uint64_t* acc_full = empty + PF_STAGES;                   // [2]
  uint64_t* acc_empty = acc_full + 2;                       // [2], waited on in the leader only
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd = abort + 1;               // not zero: some tile of this CTA has a factor that is no float (fp8.cuh)
  const RowTables tables = row_tables_at(base + PF_BARS, p.experts);
  uint8_t* turn = base + ((PF_BARS + row_tables_bytes(p.experts) + 1023) & ~1023);
  uint8_t* tiles = turn + PF_SUMS * PF_TURN;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cluster_rank = pair_rank(), rank = cluster_rank & 1u, leader = cluster_rank & ~1u;
  const int split = SPLIT ? p.split : 1, share = SPLIT ? (int)(cluster_rank >> 1) : 0;
  const int pair = (int)blockIdx.x / (2 * split), pairs = (int)gridDim.x / (2 * split);
  const int g0 = p.groups * share / split, g1 = p.groups * (share + 1) / split;
  const int w_rows = (GATED ? 2 : 1) * p.features;

  if (threadIdx.x == 0) {
    for (int s = 0; s < PF_STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full + a, 1);
      mbar_init(acc_empty + a, 2 * PF_SUMS);   // one arrival per warp of both CTAs' sums
    }
    mbar_init(drain, 1);
    *odd = 0;
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  pair_sync();                                 // the peer's barriers exist before anything lands
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bf_pdl_wait();
  fill_row_tables(tables, p.starts, p.experts, p.rows, PF_TILE);
  __syncthreads();
  const int units = tables.before[p.experts] * p.tiles_f;
  int next = 0;                                // (copying thread) the stage behind its last fill
  uint32_t next_phase = 0;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == 0) {
      // --------------------------------------------------------------- copies
      if (lane == 0) {
        const uint32_t full_leader = pair_map(smem_u32(full), leader);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = pair; u < units && ok && !*abort; u += pairs) {
          const RowTile t = row_tile(tables, p.experts, p.tiles_f, PF_TILE, u);
          for (int g = g0; g < g1; ++g) {
            if (!mbar_wait(empty + stage, phase ^ 1, abort)) {
              ok = false;
              break;
            }
            uint8_t* dst = tiles + (size_t)stage * PF_STAGE;
            const uint32_t bar = full_leader + 8u * (uint32_t)stage;
            if (rank == 0) mbar_expect_tx(full + stage, 2u * (uint32_t)PF_STAGE);
            pair_tma_load(dst, &map_x, bar, g * FK, t.row0 + (int)rank * 128);
            if (GATED) {
              const int o = t.expert * w_rows + t.ft * 128 + (int)rank * 64;
              pair_tma_load(dst + PF_HALF, &map_w, bar, g * FK, o);
              pair_tma_load(dst + PF_HALF + PF_HALF / 2, &map_w, bar, g * FK, o + p.features);
            } else {
              pair_tma_load(dst + PF_HALF, &map_w, bar, g * FK,
                            t.expert * w_rows + t.ft * PF_TILE + (int)rank * 128);
            }
            if (++stage == PF_STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
        next = stage;
        next_phase = phase;
        // every arrival that the leader's commits send to this CTA's barriers lands before it ends
        for (int s = 0; s < PF_STAGES && ok && !*abort; ++s) {
          ok = mbar_wait(empty + stage, phase ^ 1, abort);
          if (++stage == PF_STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------- products
      if (rank == 0) {
        const uint32_t idesc = fp8_idesc(PF_TILE, 256), elected = elect_one(), both = 3u << leader;
        int stage = 0, buf = 0;
        uint32_t phase = 0, buf_phase = 0;
        bool ok = true, seen = false;                         // a look at the next group's tiles
        for (int u = pair; u < units && ok; u += pairs) {
          for (int g = g0; g < g1; ++g) {
            if (!mbar_seen_or_wait_warp(seen, full + stage, phase, abort) ||
                !mbar_wait_warp(acc_empty + buf, buf_phase ^ 1, abort)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(tiles + (size_t)stage * PF_STAGE);
            const uint64_t a_desc = umma_desc_k_sw128(a_addr);
            const uint64_t b_desc = umma_desc_k_sw128(a_addr + PF_HALF);
#pragma unroll
            for (int k = 0; k < FK / 32; ++k)
              pair_umma_fp8(tmem_base + (uint32_t)(buf * 256), a_desc + (uint64_t)(2 * k),
                            b_desc + (uint64_t)(2 * k), idesc, k > 0 ? 1u : 0u, elected);
            pair_commit_by(acc_full + buf, both, elected);
            pair_commit_by(empty + stage, both, elected);
            if (++stage == PF_STAGES) {
              stage = 0;
              phase ^= 1;
            }
            if (++buf == 2) {
              buf = 0;
              buf_phase ^= 1;
            }
            seen = mbar_look(full + stage, phase);
          }
        }
      }
    }
    if (warp >= 2) {
      // ------------------------------------------------- factors that are no floats
      // Two warps that have nothing else to do look for them: the scales of a tile's rows (64 rows a warp) times
      // those of its two blocks of the weight (SPLIT: of this pair's groups; the others of the cluster are told).
      bool any = false;
      for (int u = pair; u < units; u += pairs) {
        const RowTile t = row_tile(tables, p.experts, p.tiles_f, PF_TILE, u);
        const int row = t.row0 + (int)rank * 128 + (warp & 1) * 64 + lane;
        const float *s0 = p.sx + min(row, t.row_end - 1), *s1 = p.sx + min(row + 32, t.row_end - 1);
        const float* w0 = p.sw + ((long long)t.expert * (GATED ? 2 : 1) * p.w_blocks + (GATED ? t.ft : t.ft * 2)) * p.groups;
        const float* w1 = w0 + (GATED ? (long long)p.w_blocks : t.ft * 2 + 1 < p.w_blocks ? 1LL : 0LL) * p.groups;
        for (int first = g0; first < g1; first += 32) {
          const int n = min(32, g1 - first);
          const float a = w0[first + min(lane, n - 1)], b = w1[first + min(lane, n - 1)];
          uint32_t note = 0u;
#pragma unroll 4
          for (int i = 0; i < n; ++i) {
            const float wa = __shfl_sync(0xffffffffu, a, i), wb = __shfl_sync(0xffffffffu, b, i);
            const float x0 = s0[(first + i) * p.lds], x1 = s1[(first + i) * p.lds];
            note = max(max(fp8_note(x0 * wa), fp8_note(x0 * wb)), note);
            note = max(max(fp8_note(x1 * wa), fp8_note(x1 * wb)), note);
          }
          if (__any_sync(0xffffffffu, note >= FP8_ODD))
            for (int i = 0; i < n; ++i) {
              const float wa = __shfl_sync(0xffffffffu, a, i), wb = __shfl_sync(0xffffffffu, b, i);
              const float x0 = s0[(first + i) * p.lds], x1 = s1[(first + i) * p.lds];
              any = any || fp8_odd(x0, wa) || fp8_odd(x0, wb) || fp8_odd(x1, wa) || fp8_odd(x1, wb);
            }
        }
      }
      if (any)
        for (int q = 0; q < split; ++q)
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                           pair_map(smem_u32(const_cast<int*>(odd)), (SPLIT ? 2u * (uint32_t)q : leader) + rank)),
                       "r"(1)
                       : "memory");
    }
    if (SPLIT) {
      __syncwarp();
      pair_sync();                               // the ring is free in every CTA
      pair_sync();                               // every part is in place
    }
    if (warp >= 2) named_sync(1, (PF_SUMS + 2) * 32);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    // ----------------------------------------------------------------- sums
    // A warp's 64 columns: neighbours, or (gated) the gate rows' and the up rows' of 32 outputs.
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    const int col_a = GATED ? (part >> 1) * 128 + (part & 1) * 32 : part * 64;
    const int col_b = col_a + (GATED ? 64 : 32);
    const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t acc_empty_leader = pair_map(smem_u32(acc_empty), leader);
    bool met = false;                          // (SPLIT) the cluster's two barriers are behind
    uint8_t* my_turn = turn + (warp - 4) * PF_TURN;
    const bool vec = ((uintptr_t)out & 15) == 0 && p.ldo * (int)sizeof(OutT) % 16 == 0;
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int u = pair; u < units; u += pairs) {
      const RowTile t = row_tile(tables, p.experts, p.tiles_f, PF_TILE, u);
      const int row_w0 = t.row0 + (int)rank * 128 + quarter * 32;      // the warp's first row
      const int row = min(row_w0 + lane, t.row_end - 1);               // (rows behind the last are not stored)
      const float* sx = p.sx + (long long)g0 * p.lds + row;
      // plain: the columns lie in one block of 128 weight rows; gated: in a gate's and an up's
      const long long block = (long long)t.expert * (GATED ? 2 : 1) * p.w_blocks;
      const float* swa =
          p.sw + (block + (GATED ? t.ft : min(t.ft * 2 + (part >> 1), p.w_blocks - 1))) * p.groups + g0;
      const long long to_b = GATED ? (long long)p.w_blocks * p.groups : 0;
      float acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0.f;
      bool ok = true;
      float s = *sx, wa = *swa, wb = GATED ? swa[to_b] : 0.f;
      for (int g = g0; g < g1; ++g) {
        const float fa = fp8_loop_factor(s, wa), fb = GATED ? fp8_loop_factor(s, wb) : fa;
        if (g + 1 < g1) {                                    // the next group's, under this one's wait
          sx += p.lds;
          ++swa;
          s = *sx;
          wa = *swa;
          if (GATED) wb = swa[to_b];
        }
        if (!mbar_wait_warp(acc_full + buf, buf_phase, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t r[16];
          tmem_ld16(taddr + (uint32_t)(buf * 256 + (c < 32 ? col_a + c : col_b + c - 32)), r);
          if (c == 48) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) pair_arrive_relaxed(acc_empty_leader + 8u * (uint32_t)buf);
          }
          const float f = c < 32 ? fa : fb;
#pragma unroll
          for (int j = 0; j < 16; j += 2) fma2v(acc[c + j], acc[c + j + 1], r[j], r[j + 1], f, f);
        }
        if (++buf == 2) {
          buf = 0;
          buf_phase ^= 1;
        }
      }
      bool mine = true;                                      // to store
      if constexpr (SPLIT) {
        // part p's 64 columns belong to pair p split / 4: [sender][four columns][row][4]
        const int owner = split == 4 ? part : part >> 1, slice4 = 64 / split, first4 = split == 4 ? 0 : (part & 1) * 16;
        const int lane_row = quarter * 32 + lane;
        pair_sync();                                         // the ring is free in every CTA
        mine = owner == share;
        if (!mine) {
          const int slot = share < owner ? share : share - 1;
          const uint32_t to = pair_map(smem_u32(tiles) + (uint32_t)(((slot * slice4 + first4) * 128 + lane_row) * 16),
                                       (uint32_t)(2 * owner) + rank);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (uint32_t)(j * 128 * 16)),
                         "f"(acc[4 * j]), "f"(acc[4 * j + 1]), "f"(acc[4 * j + 2]), "f"(acc[4 * j + 3])
                         : "memory");
        }
        pair_sync();                                         // every part is in place
        met = true;
        if (mine) {
          // (this pair's own part first, then the others' in their order)
          for (int slot = 0; slot < split - 1; ++slot) {
            const uint8_t* from = tiles + ((slot * slice4 + first4) * 128 + lane_row) * 16;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float4 v = *reinterpret_cast<const float4*>(from + j * 128 * 16);
              acc[4 * j] += v.x;
              acc[4 * j + 1] += v.y;
              acc[4 * j + 2] += v.z;
              acc[4 * j + 3] += v.w;
            }
          }
        }
      }
      if (!ok) break;
      const float w = p.row_w ? p.row_w[row] : 1.f;
      const int n_rows = t.row_end - row_w0;
      if (n_rows > 0 && mine) {
        OutT* dst = out + (long long)row_w0 * p.ldo;
        constexpr int COLS = 64 / (int)sizeof(OutT);         // of 64 bytes
#pragma unroll
        for (int c = 0; c < (GATED ? 32 : 64); c += COLS) {
          const int o = GATED ? t.ft * 128 + part * 32 : t.ft * PF_TILE + part * 64 + c;
          uint4 v[4];
          uint32_t* v32 = reinterpret_cast<uint32_t*>(v);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if constexpr (GATED)
              v32[j] = pack_bf16x2(
                  __float_as_uint(w * fp8_gate(p.act, acc[2 * j], acc[32 + 2 * j], p.gk)),
                  __float_as_uint(w * fp8_gate(p.act, acc[2 * j + 1], acc[33 + 2 * j], p.gk)));
            else if constexpr (sizeof(OutT) == 4)
              v32[j] = __float_as_uint(w * acc[c + j]);
            else
              v32[j] = pack_bf16x2(__float_as_uint(w * acc[c + 2 * j]), __float_as_uint(w * acc[c + 2 * j + 1]));
          }
          if (o < p.features)
            turn_and_store<OutT>(my_turn, v, dst + o, p.ldo, n_rows, p.features - o, vec, lane);
        }
      }
    }
    if (SPLIT && !met) {
      pair_sync();
      pair_sync();
    }
    named_sync(1, (PF_SUMS + 2) * 32);
    if (*odd && !*abort) {
      // (rare) Results with such factors anew, over what the warp has stored.  A thread has its row of the warp's tiles;
      // the weight's rows that the warp's columns are lie in one block, or (gated) in two.
      for (int u = pair; u < units; u += pairs) {
        const RowTile t = row_tile(tables, p.experts, p.tiles_f, PF_TILE, u);
        const int row = t.row0 + (int)rank * 128 + quarter * 32 + lane;
        const int o0 = GATED ? t.ft * 128 + part * 32 : t.ft * PF_TILE + part * 64;
        if (row >= t.row_end || o0 >= p.features || (SPLIT && (split == 4 ? part : part >> 1) != share)) continue;
        const uint8_t* xr = p.x + (size_t)row * p.ldx16 * 16;
        const float* swa = p.sw + ((long long)t.expert * (GATED ? 2 : 1) * p.w_blocks + (o0 >> 7)) * p.groups;
        auto scale_x = [&](int g) { return p.sx[g * p.lds + row]; };
        auto scale_w = [&](int up) {
          return [at = swa + (long long)up * p.w_blocks * p.groups](int g) { return at[g]; };
        };
        auto x_at = [&](int g, int k) { return xr + g * FK + k; };
        auto sum = [&](int o, int up) {
          const uint8_t* wr = p.w + ((size_t)t.expert * w_rows + up * p.features + o) * p.ldw16 * 16;
          return fp8_sum_anew(
              0, p.groups, p.K, scale_x, scale_w(up), x_at, [&](int g, int k) { return wr + g * FK + k; });
        };
        if (!fp8_any_odd(0, p.groups, p.K, scale_x, scale_w(0), x_at) &&
            (!GATED || !fp8_any_odd(0, p.groups, p.K, scale_x, scale_w(1), x_at)))
          continue;
        const float w = p.row_w ? p.row_w[row] : 1.f;
        for (int o = o0; o < min(o0 + (GATED ? 32 : 64), p.features); ++o)
          bf_st(out + (long long)row * p.ldo + o,
                w * (GATED ? fp8_gate(p.act, sum(o, 0), sum(o, 1), p.gk) : sum(o, 0)));
      }
    }
  }

  // ------------------------------------------------------------------ wind-down
  __syncthreads();
  if (*abort) {
    if (threadIdx.x == 0) {
      atomicOr(p.err, BF_ERR_WAIT);
      // the peer leaves its waits at once instead of running each of them out
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                       pair_map(smem_u32(const_cast<int*>(abort)), cluster_rank ^ 1u)),
                   "r"(1)
                   : "memory");
    }
    if (warp == 0 && lane == 0 && rank == 0) mbar_drain(full, PF_STAGES, next, next_phase);
    if (warp == 1 && rank == 0) {
      pair_commit_own(drain);
      const long long t0 = clock64();
      while (!mbar_try_wait(drain, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES / 16) {
      }
    }
    __syncthreads();
  }
  tc_fence_before();
  pair_sync();                                 // neither CTA's memory goes while the other uses it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512)
                 : "memory");
  }
}

template <typename OutT, bool GATED, bool SPLIT>
int pair_launch(const void* x, long long ldx, const void* w, long long ldw, OutT* out, PairParams p,
                int num_sms, cudaStream_t stream) {
  p.tiles_f = (p.features + (GATED ? 127 : PF_TILE - 1)) / (GATED ? 128 : PF_TILE);
  p.w_blocks = (p.features + 127) / 128;
  p.groups = (p.K + FK - 1) / FK;
  p.x = (const uint8_t*)x;
  p.w = (const uint8_t*)w;
  p.ldx16 = (uint32_t)(ldx / 16);
  p.ldw16 = (uint32_t)(ldw / 16);
  const long long tiles_r = (p.rows + PF_TILE - 1) / PF_TILE;
  const long long units = tiles_r * p.experts * p.tiles_f;
  if (units > 0x7fffffffLL || (long long)p.experts * (GATED ? 2 : 1) * p.features > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const size_t smem =
      1024 + ((PF_BARS + row_tables_bytes(p.experts) + 1023) & ~1023) + PF_SUMS * PF_TURN + (size_t)PF_STAGES * PF_STAGE;
  const size_t smem_max =
      1024 + ((PF_BARS + row_tables_bytes(FP8_MAX_EXPERTS) + 1023) & ~1023) + PF_SUMS * PF_TURN +
      (size_t)PF_STAGES * PF_STAGE;
  auto kern = fp8_pair_kernel<OutT, GATED, SPLIT>;
  static bool configured_on[BF_MAX_DEVICES];
  bool& configured = configured_on[bf_current_device()];
  if (!configured) {
    const cudaError_t ce =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_max);
    if (ce != cudaSuccess) return (int)ce;
    configured = true;
  }
  CUtensorMap mx, mw;
  int e;
  if ((e = fp8_map(&mx, x, p.rows, p.K, ldx, 128)) ||
      (e = fp8_map(&mw, w, (long long)p.experts * (GATED ? 2 : 1) * p.features, p.K, ldw, GATED ? 64 : 128)))
    return e;
  if (SPLIT && (p.starts || units * 2 * p.split > num_sms || p.groups < p.split)) return (int)cudaErrorInvalidValue;
  const long long pairs = SPLIT ? units * p.split : units < num_sms / 2 ? units : num_sms / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(PF_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = bf_pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = SPLIT ? 2 * p.split : 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t ce = cudaLaunchKernelEx(&cfg, kern, mx, mw, out, p);
  if (ce != cudaSuccess) return (int)ce;
  return bf_launch_status();
}

}  // namespace

// Arguments as bf_gemm_fp8_few's; split: pairs that share a tile, 1, 2 or 4 (without experts, where tiles * 2 *
// split is at most num_sms and there are as many groups; else 1 is taken).
BF_EXPORT int bf_gemm_fp8_pair(const void* x, long long ldx, const float* sx, long long lds, const void* w,
                               long long ldw, const float* sw, const int* starts, const float* row_w,
                               void* out, long long ldo, int out_dtype, int rows, int features, int K,
                               int experts, int gated, int act, float limit, float slope, float up_offset,
                               int split, int num_sms, int* err, cudaStream_t stream) {
  if (rows <= 0 || features <= 0) return 0;
  if (K <= 0 || experts < 1 || experts > FP8_MAX_EXPERTS || (!starts && experts != 1) || ldx % 16 || ldw % 16 ||
      ldx >> 35 || ldw >> 35 || (((uintptr_t)x | (uintptr_t)w) & 15) || num_sms < 2 ||
      (act != BF_ACT_SILU && act != BF_ACT_CLAMPED) || (gated && out_dtype != BF_DTYPE_BF16))
    return (int)cudaErrorInvalidValue;
  PairParams p = {};
  p.rows = rows;
  p.features = features;
  p.K = K;
  p.experts = experts;
  p.starts = starts;
  p.sx = sx;
  p.lds = lds;
  p.sw = sw;
  p.row_w = row_w;
  p.ldo = ldo;
  p.act = act;
  p.gk = BfGateConst{limit, slope, up_offset};
  p.err = err;
  const long long tiles = (rows + 255LL) / 256 * ((features + (gated ? 127 : 255)) / (gated ? 128 : 256));
  p.split = split == 2 || split == 4 ? split : 1;
  if (starts || tiles * 2 * p.split > num_sms || p.split > (K + FK - 1) / FK) p.split = 1;
  auto go = [&](auto* o, auto is_gated) {
    using T = std::remove_pointer_t<decltype(o)>;
    constexpr bool G = decltype(is_gated)::value;
    return p.split > 1 ? pair_launch<T, G, true>(x, ldx, w, ldw, o, p, num_sms, stream)
                       : pair_launch<T, G, false>(x, ldx, w, ldw, o, p, num_sms, stream);
  };
  if (gated) return go((__nv_bfloat16*)out, std::true_type{});
  if (out_dtype == BF_DTYPE_F32) return go((float*)out, std::false_type{});
  return go((__nv_bfloat16*)out, std::false_type{});
}
