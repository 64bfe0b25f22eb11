// Products with weights in 8 bits for few rows a weight: out[m, n] = sum_t sx[m, t] sw[n / 128, t]
// sum_{k in t} cx[m, k] cw[n, k] over the groups t of 128 columns (the format: fp8.cuh).
//
// The weight's rows are the product's rows (128 of them = 128 lanes of tensor memory) and the
// activations' rows its columns, of which a tile has as many as there are, rounded up to 16: nothing is
// multiplied for rows that are not there, and an expert with 37 rows pays for 48.  One
// tcgen05.mma.kind::f8f6f4 takes K = 32; the four of a group go into columns of tensor memory of their own,
// a ring of them, and the epilogue's warps add each group's sums, times its two scales, into registers
// (float; the scales cannot ride along in tensor memory).
//
//   warp 0       TMA: 128 weight rows and NB activation rows x 128 bytes per stage
//   warp 1       the products; TMEM allocation
//   warp 2       the factors sx sw of every column of a group, into shared memory; whether one is no float (fp8.cuh)
//   warps 4-11   the sums, times the factors, into registers; the result
//
// What bounds it with few rows is the weights' bytes (8 rows, 24,576 x 4,096 gated: 21.2 us with the rows'
// codes, 4.8 TB/s) or, of narrow weights, the way from the last of them to the end: a group passes 350
// cycles of the issuing warp and 230 and more of the sums', the parts of a cluster meet in 1 us (4,096 x 4,096:
// 8.7 us, of which 1.0 are the rows' codes).  A tile is 128 rows of the weight, so that a narrow weight alone does
// not give every SM work: then a cluster of `split` CTAs shares a tile, each a part of the groups, and the
// parts meet in shared memory, added in the order of the ranks.
// With more rows it is what a group costs beside its products (157 rows, 6,144 x 4,096: 17 us; the tensor
// pipe is busy 4 % of the time at 8 rows).  The factors come by broadcast loads from shared memory, of which an
// SM takes 128 bytes a cycle: with tiles of 128 columns that was the bound (1,030 cycles a group), so 64 is the most.
// With experts the tiles are dealt out to persistent CTAs.
//
// RESIDENT: at most eight rows come as bfloat16, and every CTA puts its columns of them into 8 bits by
// itself (warps 4-11, before the first sums, while the first weights are on their way), where they stay:
// no kernel in front, nothing of them through global memory.
//
// Every wait is bounded; no load uses multicast.
#include "common.cuh"
#include "fp8.cuh"
#include "fp8_umma.cuh"

namespace {

constexpr int FEW_THREADS = 384;
constexpr int FEW_MAX_STAGES = 12;
constexpr int FEW_BARS = 1024;
// RESIDENT: rows, and turns in which the CTA puts its columns of them into 8 bits (32 groups each).  A turn is
// 0.6 us, a kernel in front 1.6 with its way from end to start: within a graph the two come out alike (one row,
// 4,096 x 2,048 to 12,288: 7.1 to 12.7 us so and 7.0 to 12.6 with it, 1,024 x 2,048: 4.5 and 5.0), one by one 4 us of
// the host's time are gained at every size.  With more turns the kernel in front is faster.
constexpr int FEW_RES_ROWS = 8;
constexpr int FEW_ROUNDS = 4;
constexpr int FEW_W_BYTES = 128 * FK;
// Two CTAs share an SM: its registers, its shared memory and its tensor memory are dealt out by halves.  A
// step of eight rows against 24,576 x 4,096 gated took 27.5 us with one, whose 192 tiles ran in two turns.
// With 256 columns of tensor memory each (umma_utils.cuh: why no more, and no less shared memory than 92 KB).
constexpr int FEW_PER_SM = 2;
constexpr size_t FEW_SMEM = 112 * 1024;
static_assert(FEW_PER_SM * (FEW_SMEM + SMEM_OWN) <= SMEM_SM, "resident together");
constexpr int FEW_DOES_NOT_FIT = -1;

template <int NB>
struct FewShape {
  static constexpr int SLOTS = 256 / NB < 16 ? 256 / NB : 16;      // groups in tensor memory
  static constexpr int CH = NB == 16 ? 8 : 16;                     // columns a warp reads at once
  // the up rows' sums on their way to the gate rows' warps: two buffers for each half of the warps
  static constexpr int EXCHANGE = 2 * 2 * CH * 64 * 4;
};

struct FewParams {
  int rows, features, K, groups;
  int experts, tiles_f, w_blocks;      // w_blocks: rows of scales of a matrix
  const int* starts;                   // null: no experts
  const float* sx;                     // [groups, lds]
  long long lds;
  const float* sw;                     // [experts * (gated ? 2 : 1) * w_blocks, groups]
  const float* row_w;                  // per row, or null
  int split, stages, table_bytes;
  const uint8_t *codes, *w;            // what the tensor maps show
  long long ldw;
  const __nv_bfloat16* x;              // RESIDENT: the rows, res_groups groups of each in a CTA
  long long ldx;
  int x_vec, res_groups;
  long long ldo;
  int act;
  BfGateConst gk;
  int* err;
};

__device__ __forceinline__ uint32_t few_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t few_map(uint32_t local_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local_addr), "r"(rank));
  return r;
}

template <int NB, typename OutT, bool GATED, bool RESIDENT>
__global__ void __launch_bounds__(FEW_THREADS, FEW_PER_SM)
fp8_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
               OutT* __restrict__ out, const FewParams p) {
  constexpr int SLOTS = FewShape<NB>::SLOTS, CH = FewShape<NB>::CH, CHUNKS = NB / CH / 2;
  constexpr int STAGE = FEW_W_BYTES + (RESIDENT ? 0 : NB * FK);
  constexpr int HALVES = GATED ? 2 : 1;
  constexpr int TMEM_COLS = SLOTS * NB;
  static_assert(TMEM_COLS * FEW_PER_SM <= TMEM_SM_COLS, "none waits for the other's tensor memory");
  extern __shared__ __align__(16) uint8_t smem_raw[];
  BF_TRACE_POINT(10 * BF_TR_FP8_GEMM);
  bf_pdl_trigger();
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(base);
  uint64_t* empty = full + FEW_MAX_STAGES;
  uint64_t* acc_full = empty + FEW_MAX_STAGES;           // [SLOTS]: the sums and the factors are there
  uint64_t* acc_empty = acc_full + SLOTS;
  uint64_t* drain = acc_empty + SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* factors = reinterpret_cast<float*>(base + FEW_BARS);            // [SLOTS][HALVES][NB]
  // whether a factor was no float (fp8.cuh): of all tiles, the cluster's; RESIDENT: of this CTA's part of the tile
  volatile int* odd = reinterpret_cast<volatile int*>(factors + SLOTS * HALVES * NB);
  float* exchange = factors + SLOTS * HALVES * NB + 16;  // gated: up sums; split: the parts sent here
  uint8_t* table_smem = reinterpret_cast<uint8_t*>(exchange) +
                        (p.split > 1 ? ((NB + p.split - 1) / p.split) * p.split * 128 * 4
                                     : GATED ? FewShape<NB>::EXCHANGE : 0);
  const RowTables tables = row_tables_at(table_smem, p.experts);
  uint64_t* ready = drain + 2;                           // [FEW_ROUNDS]
  float* res_sx = reinterpret_cast<float*>(table_smem + p.table_bytes);        // [res_groups][NB]
  uint8_t* res = base + (((table_smem - base) + p.table_bytes + (RESIDENT ? p.res_groups * NB * 4 : 0) + 1023) & ~1023);
  uint8_t* tiles = res + (RESIDENT ? p.res_groups * FEW_RES_ROWS * FK : 0);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? (int)few_rank() : 0;
  const int cluster = (int)blockIdx.x / p.split, clusters = (int)gridDim.x / p.split;
  const int g0 = (int)((long long)p.groups * rank / p.split);
  const int g1 = (int)((long long)p.groups * (rank + 1) / p.split);
  const int STAGES = p.stages;
  const int w_rows = HALVES * p.features;                // of an expert
  // RESIDENT: 32 places of eight lanes, a row and group each: so many groups a turn
  int row_shift = 0;
  while (RESIDENT && (1 << row_shift) < p.rows) ++row_shift;
  const int per_round = 32 >> row_shift;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int a = 0; a < SLOTS; ++a) {
      mbar_init(acc_full + a, 2);              // the products' commit, the factors' warp
      mbar_init(acc_empty + a, 8);             // a warp of the epilogue each
    }
    for (int r = 0; RESIDENT && r * per_round < g1 - g0; ++r) mbar_init(ready + r, 8);
    mbar_init(drain, 1);
    if (!p.starts) {                           // (all rows are one expert's: nothing of the stream to wait for)
      tables.first[0] = 0;
      tables.end[0] = p.rows;
      tables.before[0] = 0;
      tables.before[1] = (p.rows + NB - 1) / NB;
    }
    *abort = 0;
    *odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // A group's rows of the weight: one box, or (gated) the gate rows' and the up rows'.
  constexpr int BOX = GATED ? 64 : 128;
  auto first_row = [&](int expert, int ft, int half) { return expert * w_rows + half * p.features + ft * BOX; };
  // (clusters: nothing goes to a CTA that has not begun)
  if (p.split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // Without experts a ring's worth of the weight goes into L2 before the wait for the kernels ahead.  No further: one
  // of those may be writing it (a weight is made, or written to, like any tensor).
  if (warp == 0 && lane == 0 && !p.starts) {
    const int ft = cluster / ((p.rows + NB - 1) / NB);
    for (int g = g0; g < min(g0 + STAGES, g1); ++g)
#pragma unroll
      for (int h = 0; h < HALVES; ++h) tma_prefetch_2d(&map_w, g * FK, first_row(0, ft, h));
  }
  __syncwarp();
  bf_pdl_wait();
  BF_TRACE_POINT(10 * BF_TR_FP8_GEMM + 1);
  if (p.split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (p.starts) {
    fill_row_tables(tables, p.starts, p.experts, p.rows, NB);
    __syncthreads();
  }
  const int units = tables.before[p.experts] * p.tiles_f;

  int stage = 0;                                 // of this role, with its phase
  uint32_t phase = 0;
  if (warp == 0) {
    // --------------------------------------------------------------- copies
    if (lane == 0) {
      bool ok = true;
      for (int u = cluster; u < units && ok && !*abort; u += clusters) {
        const RowTile t = row_tile(tables, p.experts, p.tiles_f, NB, u);
        for (int g = g0; g < g1; ++g) {
          if (!mbar_wait(empty + stage, phase ^ 1, abort)) {
            ok = false;
            break;
          }
          mbar_expect_tx(full + stage, STAGE);
          uint8_t* dst = tiles + (size_t)stage * STAGE;
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tma_load_2d(dst + h * BOX * FK, &map_w, full + stage, g * FK, first_row(t.expert, t.ft, h));
          if (!RESIDENT) tma_load_2d(dst + FEW_W_BYTES, &map_x, full + stage, g * FK, t.row0);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- products
    const uint32_t elected = elect_one();
    int slot = 0;
    uint32_t slot_phase = 0;
    bool ok = true, seen_empty = true, seen_full = false;        // looks at the next group's barriers
    int slots_left = SLOTS;                                      // never used so far: nothing to wait for
    const int tiles_mine = cluster < units ? (units - cluster + clusters - 1) / clusters : 0;
    int refills = tiles_mine * (g1 - g0) - STAGES;               // stages that will be filled again
    for (int u = cluster; u < units && ok; u += clusters) {
      const RowTile t = row_tile(tables, p.experts, p.tiles_f, NB, u);
      const int n = min(NB, (t.row_end - t.row0 + 15) & ~15);
      const uint32_t idesc = fp8_idesc(128, n);
      for (int g = g0; g < g1; ++g) {
        if (!mbar_seen_or_wait_warp(slots_left > 0 || seen_empty, acc_empty + slot, slot_phase ^ 1, abort) ||
            !mbar_seen_or_wait_warp(seen_full, full + stage, phase, abort) ||
            (RESIDENT && !mbar_wait_warp(ready + (g - g0) / per_round, 0, abort))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(tiles + (size_t)stage * STAGE), d_tmem = tmem_base + (uint32_t)(slot * NB);
        const uint64_t a_desc = umma_desc_k_sw128(a_addr);
        const uint64_t b_desc =
            // (eight rows: the product's second eight columns read them again)
            RESIDENT ? umma_desc_k_sw128_sbo(smem_u32(res + (g - g0) * FEW_RES_ROWS * FK), 0u)
                     : umma_desc_k_sw128(a_addr + FEW_W_BYTES);
        uint64_t* const done_stage = empty + stage;
        uint64_t* const done_slot = acc_full + slot;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
        if (++slot == SLOTS) {
          slot = 0;
          slot_phase ^= 1;
        }
        if (--slots_left <= 0) seen_empty = mbar_look(acc_empty + slot, slot_phase ^ 1);
        seen_full = mbar_look(full + stage, phase);
#pragma unroll
        for (int k = 0; k < FK / 32; ++k)
          umma_fp8(d_tmem, a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k), idesc, k > 0 ? 1u : 0u, elected);
        umma_commit_by(done_slot, elected);
        if (refills-- > 0) umma_commit_by(done_stage, elected);
      }
    }
  } else if (warp == 2) {
    // -------------------------------------------------------------- factors
    // The scales of AHEAD groups are asked for while the factors of the AHEAD before them are written:
    // a load takes longer than a group's products.
    constexpr int PER = (NB + 31) / 32;          // columns a lane looks after
    constexpr int AHEAD = NB <= 32 ? 8 : 4;
    int slot = 0, slots_left = SLOTS;
    uint32_t slot_phase = 0;
    bool ok = true;
    float sx[AHEAD][PER], sw[AHEAD][HALVES];
    auto scale_x = [&](const RowTile& t, int g, int j) {       // of column j * 32 + lane
      const int row = t.row0 + j * 32 + lane;
      if (RESIDENT) return row < t.row_end ? res_sx[(g - g0) * NB + row] : 1.f;
      return row < t.row_end && j * 32 + lane < NB ? p.sx[(long long)g * p.lds + row] : 1.f;
    };
    auto scale_w = [&](const RowTile& t, int g, int h) {
      const long long block = (long long)t.expert * HALVES * p.w_blocks + (GATED ? t.ft >> 1 : t.ft);
      return p.sw[(block + h * p.w_blocks) * p.groups + g];
    };
    auto ask = [&](const RowTile& t, int ga) {
      if (RESIDENT) ok = mbar_wait_warp(ready + (min(ga + AHEAD, g1) - 1 - g0) / per_round, 0, abort);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int g = min(ga + i, g1 - 1);
#pragma unroll
        for (int j = 0; j < PER; ++j) sx[i][j] = scale_x(t, g, j);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) sw[i][h] = scale_w(t, g, h);
      }
    };
    int u = cluster;
    RowTile t;
    if (u < units) {
      t = row_tile(tables, p.experts, p.tiles_f, NB, u);
      ask(t, g0);
    }
    bool odd_here = false;
    for (; u < units && ok; u += clusters) {
      for (int ga = g0; ga < g1 && ok; ga += AHEAD) {
        float f[AHEAD][PER * HALVES];
        uint32_t note = 0u;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
          for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              f[i][j * HALVES + h] = fp8_loop_factor(sx[i][j], sw[i][h]);
              note = max(note, fp8_note(f[i][j * HALVES + h]));
            }
        if (__builtin_expect(note >= FP8_ODD, 0)) {
#pragma unroll 1
          for (int i = 0; i < AHEAD * PER * HALVES; ++i) {
            const int g = min(ga + i / (PER * HALVES), g1 - 1);
            odd_here = odd_here || fp8_odd(scale_x(t, g, i / HALVES % PER), scale_w(t, g, i % HALVES));
          }
        }
        if (ga + AHEAD < g1) {
          ask(t, ga + AHEAD);
        } else if (u + clusters < units) {
          t = row_tile(tables, p.experts, p.tiles_f, NB, u + clusters);
          ask(t, g0);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          if (ga + i >= g1 || !ok) break;
          if (--slots_left < 0 && !mbar_wait_warp(acc_empty + slot, slot_phase ^ 1, abort)) {
            ok = false;
            break;
          }
          float* dst = factors + slot * HALVES * NB;
#pragma unroll
          for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
              if (j * 32 + lane < NB) dst[h * NB + j * 32 + lane] = f[i][j * HALVES + h];
          if (RESIDENT && odd_here) *odd = 1;
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_full + slot);
          if (++slot == SLOTS) {
            slot = 0;
            slot_phase ^= 1;
          }
        }
      }
    }
    if (!RESIDENT && odd_here)
      for (int r = 0; r < p.split; ++r)
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                         few_map(smem_u32(const_cast<int*>(odd)), (uint32_t)r)),
                     "r"(1)
                     : "memory");
  } else if (warp >= 4) {
    // ----------------------------------------------------------------- sums
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int lane_row = quarter * 32 + lane;            // of the tile's 128 weight rows
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int which = GATED ? quarter >> 1 : 0;
    if constexpr (RESIDENT) {
      const int place = (warp - 4) * 4 + (lane >> 3), sub = lane & 7;
      const int row = place & ((1 << row_shift) - 1);
      const int rounds = (g1 - g0 + per_round - 1) / per_round;
      const __nv_bfloat16* src = p.x + row * p.ldx + sub * 16;
      auto ask = [&](int r, Fp8Sixteen<__nv_bfloat16, 8>& v) {
        const int k = (g0 + r * per_round + (place >> row_shift)) * FK;
        const int left = row < p.rows && k < g1 * FK ? p.K - k - sub * 16 : 0;
        if (p.x_vec && left >= 16) {
          v.template load<true>(src + k, 16);
        } else {
          v.template load<false>(src + k, left);
        }
      };
      Fp8Sixteen<__nv_bfloat16, 8> v, next;
      ask(0, v);
      for (int r = 0; r < rounds; ++r) {
        if (r + 1 < rounds) ask(r + 1, next);
        const int gl = r * per_round + (place >> row_shift);
        uint32_t m = v.largest();
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const Fp8Scale sc = fp8_scale(m);
        if (row < p.rows && gl < g1 - g0) {
          *reinterpret_cast<uint4*>(res + (gl * FEW_RES_ROWS + row) * FK + ((sub ^ (row & 7)) << 4)) = v.codes(sc);
          if (sub == 0) res_sx[gl * NB + row] = sc.s;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(ready + r);
        v = next;
      }
    }
    int slot = 0;
    uint32_t slot_phase = 0;
    for (int u = cluster; u < units; u += clusters) {
      const RowTile t = row_tile(tables, p.experts, p.tiles_f, NB, u);
      const int n = min(NB, t.row_end - t.row0);
      float acc[CHUNKS][CH];
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < CH; ++j) acc[i][j] = 0.f;
      bool ok = true;
      for (int g = g0; g < g1; ++g) {
        if (!mbar_wait_warp(acc_full + slot, slot_phase, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float* f = factors + (slot * HALVES + which) * NB;
        // (the two halves of the warps take the chunks in turn, one after the other: a warp has two at most)
        const uint32_t at = tmem_base + lanes + (uint32_t)(slot * NB + half * CH);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int c = (2 * i + half) * CH;
          if (c < n) {
            uint32_t r[CH];
            tmem_ask(at + (uint32_t)(2 * i * CH), r);
            tmem_got();
            tmem_have(r);
#pragma unroll
            for (int j = 0; j < CH; j += 4) {
              const float4 v = *reinterpret_cast<const float4*>(f + c + j);
              fma2v(acc[i][j], acc[i][j + 1], r[j], r[j + 1], v.x, v.y);
              fma2v(acc[i][j + 2], acc[i][j + 3], r[j + 2], r[j + 3], v.z, v.w);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty + slot);
        if (++slot == SLOTS) {
          slot = 0;
          slot_phase ^= 1;
        }
      }
      if constexpr (RESIDENT) {
        const int feature = t.ft * BOX + (lane_row & (BOX - 1));
        if (__builtin_expect(ok && *odd != 0 && feature < p.features, 0)) {
          // (rare) the sums over this CTA's groups anew
          const uint8_t* wr = p.w + ((long long)which * p.features + feature) * p.ldw;
          const float* swr = p.sw + (which * p.w_blocks + (feature >> 7)) * (long long)p.groups;
          for (int a = 0; a < CHUNKS * CH; ++a) {
            const int c = (2 * (a / CH) + half) * CH + a % CH;
            if (c >= n) continue;
            auto scale_x = [&](int g) { return res_sx[(g - g0) * NB + c]; };
            auto scale_w = [&](int g) { return swr[g]; };
            auto x_at = [&](int g, int k) {
              return res + ((g - g0) * FEW_RES_ROWS + c) * FK + (((k >> 4) ^ (c & 7)) << 4) + (k & 15);
            };
            if (!fp8_any_odd(g0, g1, p.K, scale_x, scale_w, x_at)) continue;
            const float v = fp8_sum_anew(g0, g1, p.K, scale_x, scale_w, x_at, [&](int g, int k) { return wr + g * FK + k; });
#pragma unroll
            for (int i = 0; i < CHUNKS * CH; ++i) acc[i / CH][i % CH] = i == a ? v : acc[i / CH][i % CH];
          }
        }
        __syncwarp();
      }
      if (p.split > 1) {
        // column j goes to rank j % split: [rank][its number there][weight row]
        const int per = (NB + p.split - 1) / p.split;
        const uint32_t here = smem_u32(exchange);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const int c = (2 * i + half) * CH + j;
            if (c < n) {
              const uint32_t at = here + (uint32_t)(((rank * per + c / p.split) * 128 + lane_row) * 4);
              asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(few_map(at, (uint32_t)(c % p.split))),
                           "f"(acc[i][j])
                           : "memory");
            }
          }
        break;                                           // (a cluster has one tile)
      }
      if (GATED) {
        ok = named_all(1 + half, 128, ok);
        if (!ok) break;
        float* xb = exchange + half * 2 * CH * 64;
        const int o = t.ft * 64 + (quarter & 1) * 32 + lane;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int c = (2 * i + half) * CH;
          if (c < n) {                                   // (the same in the four warps)
            float* b = xb + (i & 1) * CH * 64 + (quarter & 1) * 32 + lane;
            if (quarter >= 2) {
#pragma unroll
              for (int j = 0; j < CH; ++j) b[j * 64] = acc[i][j];
            }
            named_sync(1 + half, 128);
            if (quarter < 2 && o < p.features) {
#pragma unroll
              for (int j = 0; j < CH; ++j)
                if (c + j < n) {
                  const int row = t.row0 + c + j;
                  float v = fp8_gate(p.act, acc[i][j], b[j * 64], p.gk);
                  if (p.row_w) v *= p.row_w[row];
                  bf_st(out + (size_t)row * p.ldo + o, v);
                }
            }
          }
        }
        // (the next tile's first buffer is this tile's first too: two barriers lie between its uses
        // only if this tile had more than one chunk)
        named_sync(1 + half, 128);
      } else {
        if (!ok) break;
        const int o = t.ft * 128 + lane_row;
        if (o < p.features) {
#pragma unroll
          for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int j = 0; j < CH; ++j) {
              const int c = (2 * i + half) * CH + j;
              if (c < n) {
                const int row = t.row0 + c;
                float v = acc[i][j];
                if (p.row_w) v *= p.row_w[row];
                bf_st(out + (size_t)row * p.ldo + o, v);
              }
            }
        }
      }
    }
  }
  __syncwarp();
  BF_TRACE_POINT(10 * BF_TR_FP8_GEMM + 5);

  if (p.split > 1) {
    // every part is in place behind this; then the columns of this rank, parts in the ranks' order
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (cluster < units) {
      const RowTile t = row_tile(tables, p.experts, p.tiles_f, NB, cluster);
      const int n = min(NB, t.row_end - t.row0), per = (NB + p.split - 1) / p.split;
      const int width = GATED ? 64 : 128;
      const int mine = n > rank ? (n - rank + p.split - 1) / p.split : 0;
      for (int i = threadIdx.x; i < mine * width; i += FEW_THREADS) {
        const int o = i % width, c = i / width, row = t.row0 + c * p.split + rank;
        if (t.ft * width + o >= p.features) continue;
        float v = 0.f, up = 0.f;
        for (int r = 0; r < p.split; ++r) {
          const float* part = exchange + (r * per + c) * 128 + o;
          v += part[0];
          if (GATED) up += part[64];
        }
        if (GATED) v = fp8_gate(p.act, v, up, p.gk);
        if (p.row_w) v *= p.row_w[row];
        bf_st(out + (size_t)row * p.ldo + t.ft * width + o, v);
      }
    }
  }

  // ------------------------------------------------------------------ wind-down
  __syncthreads();
  if (!RESIDENT && __builtin_expect(*odd != 0 && !*abort, 0)) {
    // (rare) results with a factor that is no float anew, over what this CTA has stored
    constexpr int WIDTH = GATED ? 64 : 128;
    for (int u = cluster; u < units; u += clusters) {
      const RowTile t = row_tile(tables, p.experts, p.tiles_f, NB, u);
      const int n = min(NB, t.row_end - t.row0);
      for (int i = threadIdx.x; i < n * WIDTH; i += FEW_THREADS) {
        const int o = t.ft * WIDTH + i % WIDTH, c = i / WIDTH, row = t.row0 + c;
        if (o >= p.features || (p.split > 1 && c % p.split != rank)) continue;
        auto scale_x = [&](int g) { return p.sx[g * p.lds + row]; };
        auto scales_w = [&](int h) {
          return p.sw + (((long long)t.expert * HALVES + h) * p.w_blocks + (o >> 7)) * p.groups;
        };
        auto x_at = [&](int g, int k) { return p.codes + row * p.ldx + g * FK + k; };
        bool any = false;
        for (int h = 0; h < HALVES; ++h)
          any = any || fp8_any_odd(0, p.groups, p.K, scale_x, [at = scales_w(h)](int g) { return at[g]; }, x_at);
        if (!any) continue;
        float v[2];
#pragma unroll 1
        for (int h = 0; h < HALVES; ++h) {
          const uint8_t* wr = p.w + ((long long)t.expert * w_rows + h * p.features + o) * p.ldw;
          const float sum = fp8_sum_anew(
              0, p.groups, p.K, scale_x, [at = scales_w(h)](int g) { return at[g]; }, x_at,
              [&](int g, int k) { return wr + g * FK + k; });
          if (h == 0) v[0] = sum; else v[1] = sum;
        }
        float r = GATED ? fp8_gate(p.act, v[0], v[1], p.gk) : v[0];
        if (p.row_w) r *= p.row_w[row];
        bf_st(out + (size_t)row * p.ldo + o, r);
      }
    }
  }
  BF_TRACE_POINT(10 * BF_TR_FP8_GEMM + 2);
  if (*abort) {
    if (threadIdx.x == 0) atomicOr(p.err, BF_ERR_WAIT);
    if (warp == 0 && lane == 0) mbar_drain(full, STAGES, stage, phase);
    if (warp == 1) {
      umma_commit(drain);
      const long long t0 = clock64();
      while (!mbar_try_wait(drain, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES / 16) {
      }
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS)
                 : "memory");
  }
}

// Shared memory in front of the ring, and the ring's stages (fewer than 2: the sizes do not fit).
template <int NB, bool GATED, bool RESIDENT>
size_t few_memory(const FewParams& p, int* stages) {
  const size_t extra = p.split > 1 ? (size_t)((NB + p.split - 1) / p.split) * p.split * 128 * 4
                                   : GATED ? FewShape<NB>::EXCHANGE : 0;
  size_t fixed = FEW_BARS + (size_t)FewShape<NB>::SLOTS * (GATED ? 2 : 1) * NB * 4 + 16 * 4 + extra + p.table_bytes;
  if (RESIDENT) fixed += (size_t)p.res_groups * NB * 4;
  fixed = 1024 + ((fixed + 1023) & ~(size_t)1023);
  if (RESIDENT) fixed += (size_t)p.res_groups * FEW_RES_ROWS * FK;
  const size_t stage = FEW_W_BYTES + (RESIDENT ? 0 : NB * FK);
  const size_t n = fixed < FEW_SMEM ? (FEW_SMEM - fixed) / stage : 0;
  *stages = n > FEW_MAX_STAGES ? FEW_MAX_STAGES : (int)n;
  const size_t all = fixed + *stages * stage;      // (93 KB at least as it is)
  return all < TMEM_LEAST_SMEM ? TMEM_LEAST_SMEM : all;
}

template <int NB, typename OutT, bool GATED, bool RESIDENT>
int few_launch(const void* x, long long ldx, const void* w, long long ldw, OutT* out, FewParams p, int num_sms,
               cudaStream_t stream) {
  auto kern = fp8_few_kernel<NB, OutT, GATED, RESIDENT>;
  static bool configured_on[BF_MAX_DEVICES];
  bool& configured = configured_on[bf_current_device()];
  if (!configured) {
    const cudaError_t ce =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SMEM);
    if (ce != cudaSuccess) return (int)ce;
    configured = true;
  }
  constexpr int HALVES = GATED ? 2 : 1;
  p.tiles_f = (p.features + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
  p.w_blocks = (p.features + 127) / 128;
  p.groups = (p.K + FK - 1) / FK;
  p.table_bytes = row_tables_bytes(p.experts);
  const long long tiles_r = (p.rows + NB - 1) / NB, room = (long long)FEW_PER_SM * num_sms;
  // (at most: `starts` may hold anything)
  const long long units = tiles_r * p.experts * p.tiles_f;
  if (units > 0x7fffffffLL || (long long)p.experts * HALVES * p.features > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  if (p.starts || units * p.split > room || p.split > p.groups) p.split = 1;
  p.codes = (const uint8_t*)x;
  p.w = (const uint8_t*)w;
  p.ldx = ldx;
  p.ldw = ldw;
  if (RESIDENT) {
    p.x = (const __nv_bfloat16*)x;
    p.x_vec = ldx % 8 == 0 && ((uintptr_t)x & 15) == 0;
    p.res_groups = (p.groups + p.split - 1) / p.split;
    int per_round = 32;
    while (32 / per_round < p.rows) per_round /= 2;
    if (p.starts || p.rows > FEW_RES_ROWS || (p.res_groups + per_round - 1) / per_round > FEW_ROUNDS) return FEW_DOES_NOT_FIT;
  }
  const size_t smem = few_memory<NB, GATED, RESIDENT>(p, &p.stages);
  if (RESIDENT && p.stages < 4) return FEW_DOES_NOT_FIT;
  if (p.stages < 2) return (int)cudaErrorInvalidValue;
  CUtensorMap mx, mw;
  int e;
  if ((e = fp8_map(&mw, w, (long long)p.experts * HALVES * p.features, p.K, ldw, GATED ? 64 : 128)) ||
      (!RESIDENT && (e = fp8_map(&mx, x, p.rows, p.K, ldx, NB))))
    return e;
  if (RESIDENT) mx = mw;                           // (not used)
  const long long work = units * p.split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.split > 1 || work < room ? work : room));
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = bf_pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  const cudaError_t ce = cudaLaunchKernelEx(&cfg, kern, mx, mw, out, p);
  if (ce != cudaSuccess) return (int)ce;
  return bf_launch_status();
}

template <typename OutT, bool GATED>
int few_by_width(int nb, bool resident, const void* x, long long ldx, const void* w, long long ldw, OutT* out,
                 const FewParams& p, int num_sms, cudaStream_t stream) {
  if (resident) {
    if (nb == 16) return few_launch<16, OutT, GATED, true>(x, ldx, w, ldw, out, p, num_sms, stream);
    return FEW_DOES_NOT_FIT;
  }
  switch (nb) {
    case 16: return few_launch<16, OutT, GATED, false>(x, ldx, w, ldw, out, p, num_sms, stream);
    case 32: return few_launch<32, OutT, GATED, false>(x, ldx, w, ldw, out, p, num_sms, stream);
    case 64: return few_launch<64, OutT, GATED, false>(x, ldx, w, ldw, out, p, num_sms, stream);
    default: return (int)cudaErrorInvalidValue;
  }
}

}  // namespace

// x codes [rows, K] (rows ldx bytes apart) with scales sx [ceil(K / 128), lds], or with `resident` bfloat16
// (rows ldx numbers apart; -1 is returned, and nothing done, where the rows do not fit); w codes [experts,
// (gated ? 2 : 1) * features, K] (rows ldw bytes apart) with scales sw [experts, (gated ? 2 : 1) *
// ceil(features / 128), ceil(K / 128)]; starts int [experts + 1] of the experts' first rows, or null for
// one weight; row_w float [rows] or null; out [rows, features], rows ldo apart.  nb: most rows of a tile
// (16, 32 or 64).  split: CTAs that share a tile (without experts, tiles * split at most 2 * num_sms, as many as
// are resident, and at most as many as there are groups; else 1 is taken).
BF_EXPORT int bf_gemm_fp8_few(const void* x, long long ldx, const float* sx, long long lds, const void* w,
                              long long ldw, const float* sw, const int* starts, const float* row_w,
                              void* out, long long ldo, int out_dtype, int rows, int features, int K,
                              int experts, int gated, int act, float limit, float slope, float up_offset,
                              int nb, int split, int resident, int num_sms, int* err,
                              cudaStream_t stream) {
  if (rows <= 0 || features <= 0) return 0;
  if (K <= 0 || experts < 1 || experts > FP8_MAX_EXPERTS || (!starts && experts != 1) || ldw % 16 ||
      ((uintptr_t)w & 15) || (!resident && (ldx % 16 || ((uintptr_t)x & 15))) || split < 1 || split > 8 || num_sms < 1 ||
      (act != BF_ACT_SILU && act != BF_ACT_CLAMPED) || (gated && out_dtype != BF_DTYPE_BF16))
    return (int)cudaErrorInvalidValue;
  FewParams p = {};
  p.rows = rows;
  p.features = features;
  p.K = K;
  p.experts = experts;
  p.starts = starts;
  p.sx = sx;
  p.lds = lds;
  p.sw = sw;
  p.row_w = row_w;
  p.split = split;
  p.ldo = ldo;
  p.act = act;
  p.gk = BfGateConst{limit, slope, up_offset};
  p.err = err;
  if (gated)
    return few_by_width<__nv_bfloat16, true>(nb, resident, x, ldx, w, ldw, (__nv_bfloat16*)out, p, num_sms, stream);
  if (out_dtype == BF_DTYPE_F32)
    return few_by_width<float, false>(nb, resident, x, ldx, w, ldw, (float*)out, p, num_sms, stream);
  return few_by_width<__nv_bfloat16, false>(nb, resident, x, ldx, w, ldw, (__nv_bfloat16*)out, p, num_sms, stream);
}

BF_TRACE_READER(bf_trace_read_gemm_fp8_few)
