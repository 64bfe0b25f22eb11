// Attention over pages held in 4 bits (layout: kv4.cuh), for rows that bring one token each and for
// prompt portions of a few rows.
//
// With k_j = m_j + s_j c_j and v_j likewise (s, m per 64 numbers, codes c of 0 to 15),
//
//   q . k_j     = sum over groups of  s_j (q . c_j) + m_j sum(q)
//   sum p_j v_j = sum over groups of  (p_j s_j) . c_j + sum p_j m_j ,
//
// so the codes go into the tensor cores as they are and scales and lowest values meet sums only.  A code
// becomes a bfloat16 operand by a mask alone: the bits 0 .. 7 of a bfloat16 number whose other bits are zero
// count steps of 2^-133 (subnormal numbers and the first binade above them), and the tensor cores take
// them as they are.  So (word & 0x000f000f) is two codes, (word & 0x00f000f0) the two beside them times 16,
// and one shift by 8 gives the other four of eight: five instructions for four operand registers.  Queries
// and probabilities carry the factor 2^64 (and 2^-4 against the codes times 16), the sums 2^69.
//
// Rounding: the probabilities times the value scales go into their product as bfloat16.  Their error meets
// the codes less 8, since 8 times the sum of the rounded products is taken off again and p (m + 8 s) added
// in float.  Everything else is float.
//
// Work.  A tile is up to 8 NT columns, a column one query head of one token row; its keys go sixteen at a
// time (a unit), for every kv head.  Every warp takes one stretch of units, fetches them by itself (16 bytes
// a lane, asynchronously, two units ahead of the two it computes) and waits for no other.  Where stretches
// are short, they are pieces of one tile and head, so that a warp begins but once; where they are long, all
// units in one row are cut into equal ones, whatever heads they cross.  A tile and head that one warp
// has whole is written by it; a cut one leaves a partial result a piece, which a second kernel adds up in
// the order of the keys: scratch is two partials a warp whatever the contexts are.  The running maximum moves
// only when a score passes it by 2^8, which no result depends on beyond rounding and which leaves one
// vote a step where maxima would take shuffles.
//
// Where there are few heads, or the tables have room for few keys only (ka_blocks_a_head), a cluster of one to
// eight blocks takes a tile and head whole: its warps leave their partials in shared memory, each block adds up its
// own and the blocks theirs over distributed shared memory, and there is no second kernel.
//
// Portions that are loaded and attended on tcgen05 leave behind which of them, and which kv heads, fp16 had no room for
// (kv4.cu): a block an SM takes those heads whole, one after the other, from the codes.  As a rule there are none, and a
// block only reads that.  Calls of 2,048 rows from position 0, 32 heads of 128 (8): 84 us with nothing noted, 232
// with one kv head, 371 with all; 256 rows behind 8,192 94, 195 and 299.  (A walk over the keys by multiply-adds took 40 and
// 85 ms.)
//
// Measured (B200), replayed in a row / with caches cold.  64 rows of 64 heads of 128 (8) behind 4,096 keys down to 2,700:
// 58.5 / 67.6 us, where the 254 MB take 39 at the rate of a copy, 6.54 TB/s.  All rows behind 2,048, 4,096, 8,192 and
// 16,384 keys: 42, 66, 114 and 208 us, so that a byte more costs what it takes at 6.3 to 6.4 TB/s and some 19 us stand
// beside the bytes: the beginning of the stretches (queries, tables, first units), a wait for the slowest SM at their end, the
// second kernel (5 to 8).  (Issue slots 48 % busy and DRAM 55 % over the attention kernel at 4,096: some 258 instructions
// a unit of 2,304 bytes are 25 us of all slots.)  Eight rows behind 4,096: clusters of two 16.4 / 20.5 (bytes: 5),
// stretches 12.5 and 3 for the second kernel; 30,000 keys behind a window of 4,096, 12 rows of 16 heads: a block a head
// 20.6 / 26.6, stretches 18 + 3 (8.7).  Tried without gain: partials added up in a block before the second kernel, barriers
// that keep a block's warps level, fewer warps with a deeper ring, the lowest values as the product's addend.
#include "common.cuh"
#include "kv4.cuh"
#include "mma_utils.cuh"

#define KA_STAGES 4                        // units: two steps
#define KA_MAX_TILES 512                   // of one launch
#define KA_UNIT 16                         // keys
#define KA_MIN_UNITS 2                     // a stretch's length at least
#define KA_LONG 24                         // units of a stretch from which heads are crossed
#define KA_PIECES 30.f                     // a head of U units gets sqrt(30 U) pieces at most
#define KA_SHARE 8                         // blocks of a cluster at most
#define KA_BEGIN 6                         // units that a warp could compute while it begins a head

// Warps of a CTA, one CTA an SM: sixteen where 128 registers hold a tile.
__host__ __device__ constexpr int ka_warps(int d, int nt) { return d <= 128 && nt == 1 ? 16 : 8; }

struct KaArgs {
  const __nv_bfloat16* q;
  long long q_stride;
  const unsigned char* cache;
  const int *rows, *seq_of_token, *positions, *items;
  int first_tile, n_tiles, tiles_per_item, T;
  const int* block_tables;
  int table_stride, table_rows, table_width;
  __nv_bfloat16* out;
  long long out_stride;
  int nh, nkv, group, chunk, chunks, tokens;               // query heads per kv head; in a tile; chunks of them
  int page_size, page_shift, num_pages, window, keep;
  float scale;
  unsigned chunk_inverse;                                  // n / chunk = n chunk_inverse >> 8 for n < 16
  int max_pieces, share, early;
  float* part_o;
  float2* part_ml;
  int4* desc;
  const int *beyond, *moved;                               // KA_AGAIN
  int n_items, heads;
  int* err;
};

// What a block of the kernel does.
enum KaForm {
  KA_STRETCHES,                            // each warp one stretch of units
  KA_HEAD,                                 // a cluster of a.share blocks takes a (tile, head) whole
  KA_AGAIN                                 // a block takes (tile, head)s whole, one after the other, of those that `beyond` notes
};

struct KaTile {
  int b, row0, pos0, ntok;
};

// Units of a tile: sixteen keys each, those of the kept first tokens, then from the window's first on.
struct KaSpan {
  int kept, from, units;
};
__device__ __forceinline__ KaSpan ka_span(const KaTile& t, int window, int keep) {
  KaSpan s = {0, 0, 0};
  if (t.ntok <= 0) return s;
  if (window > 0) {
    s.from = max(0, t.pos0 - window + 1) >> 4;
    s.kept = min((keep + KA_UNIT - 1) >> 4, s.from);
  }
  s.units = ((t.pos0 + t.ntok - 1) >> 4) - s.from + 1 + s.kept;
  static_assert(KA_UNIT == 16, "the shifts above");
  return s;
}

// a / b for 0 <= a < 2^20, 0 < b: the half keeps the product off the whole numbers by more than it is wrong
__device__ __forceinline__ int ka_div(int a, int b) { return (int)(((float)a + 0.5f) * __frcp_rn((float)b)); }
__device__ __forceinline__ float ka_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned ka_transpose(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool B>
struct Bool {
  static constexpr bool value = B;
};
__device__ __forceinline__ void ka_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A number of another block's shared memory, where this block has its own at p.
__device__ __forceinline__ float ka_peer(const float* p, int rank) {
  unsigned at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
// HEAD: the warps of the block or cluster share a head's units and add up in shared memory.
template <int D, int NT, KaForm FORM>
__global__ void __launch_bounds__(32 * ka_warps(D, NT), 1)
kv4_attention_kernel(const __grid_constant__ KaArgs a) {
  constexpr bool HEAD = FORM != KA_STRETCHES, AGAIN = FORM == KA_AGAIN;
  constexpr int NG = D / KV4_GROUP, REC = kv4_record(D), UNIT_BYTES = 2 * REC;
  constexpr int KW = D / 32, COLS = 8 * NT, WARPS = ka_warps(D, NT);
  constexpr float UP = 1.8446744073709551616e19f;           // 2^64
  constexpr float DOWN = 5.90295810358705651712e20f;        // 2^69
  constexpr unsigned M0 = 0x000f000fu, M4 = 0x00f000f0u, M8 = 0x00ff00ffu, ONES = 0x00010001u;
  extern __shared__ __align__(128) unsigned char smem[];
  KaTile* tiles = reinterpret_cast<KaTile*>(smem + (size_t)WARPS * KA_STAGES * UNIT_BYTES);
  int* units_of = reinterpret_cast<int*>(tiles + KA_MAX_TILES);            // of a head of the tile
  int* start = units_of + KA_MAX_TILES;                                    // the tile's first piece, or unit
  __shared__ int sums[WARPS];
  __shared__ float rates[WARPS];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, q4 = lane & 3;
  const int pairs = a.nkv * a.chunks;
  // Where the step's description (rows, positions, requests) was there before the kernel ahead began (a.early), it
  // is read under that kernel's end, and block tables, queries, pages and all writes wait; else everything waits.
  // The successor is asked for after the wait: its blocks, resident any earlier, slow down what runs ahead of this
  // kernel.
  auto begin = [&](int early) {
    if (early != a.early) return;
    bf_pdl_wait();
    bf_pdl_trigger();
  };
  begin(0);

  auto tile_of = [&](int id, bool flag) {
    KaTile t;
    int rows = 1, skip = 0;                                 // of the portion; before the tile
    if (a.items) {
      const int i = id / a.tiles_per_item;
      const int* it = a.items + 4 * (size_t)i;
      t.b = it[0], t.row0 = it[1], t.pos0 = it[3];
      rows = max(it[2], 0), skip = (id - i * a.tiles_per_item) * a.tokens;
    } else {
      t.row0 = a.rows ? a.rows[id] : id;
      const bool ok = t.row0 >= 0 && t.row0 < a.T;
      t.b = ok ? a.seq_of_token[t.row0] : -1;
      t.pos0 = ok ? a.positions[t.row0] : 0;
    }
    t.ntok = min(rows - skip, a.tokens);
    if (t.ntok > 0 && (t.b < 0 || t.b >= a.table_rows || t.row0 < 0 || t.row0 > a.T - rows || t.pos0 < 0 ||
                       (long long)t.pos0 + rows > (long long)a.table_width * a.page_size)) {
      if (flag) atomicOr(a.err, BF_ERR_PAGE);
      t.ntok = 0;
    }
    t.row0 += skip, t.pos0 += skip;
    return t;
  };
  const int warps = gridDim.x * WARPS;
  int me = warp, each = 1, longer = 0, x = 0, x_end = 1;
  bool aligned = true;
  if constexpr (AGAIN) {                                    // (as a rule nothing is noted)
    int any = 0;
    for (int i = tid; i < a.n_items * a.nkv; i += 32 * WARPS) any |= a.beyond[i];
    if (!__syncthreads_or(any)) return;
    x = blockIdx.x, x_end = a.heads;
  }
  if constexpr (!HEAD) {
    // ---- tiles, and how their units are cut.  (Loops, not unrolled: what a launch runs once waits for its
    // instructions most of all.)
#pragma unroll 1
    for (int e = tid; e < a.n_tiles; e += 32 * WARPS) {
      const KaTile t = tile_of(a.first_tile + e, blockIdx.x == 0);
      tiles[e] = t;
      const int n = ka_span(t, a.window, a.keep).units;
      units_of[e] = n;
    }
    __syncthreads();
    int total = 0, filled = 0, longest = 0;
#pragma unroll 1
    for (int e = lane; e < a.n_tiles; e += 32) {
      const int n = units_of[e];
      total += n, filled += n > 0, longest = max(longest, n);
    }
    total = __reduce_add_sync(0xffffffffu, total) * pairs;
    filled = __reduce_add_sync(0xffffffffu, filled) * pairs;
    longest = __reduce_max_sync(0xffffffffu, longest);
    // Short stretches: a tile's heads together get pieces in proportion to their units, one each at least.
    // With `rate` pieces a unit that makes at most rate total + heads of them: warp w tries a rate, and
    // the highest that gives every piece a warp of its own is taken.  Not too many of a head, which the second kernel
    // adds up: a head's 2,048 units in 1,024 pieces took 33 us, in 248 19.
    aligned = total < KA_LONG * warps && filled < warps;
    float rate = 0.f;
    if (aligned) {
      auto rate_of = [&](int i) {
        const float room = warps - filled * (i * (1.f / (WARPS - 1)));
        return fminf(fminf(1.f / KA_MIN_UNITS, sqrtf(KA_PIECES / longest)), fmaxf(room, 0.f) / total);
      };
      rate = rate_of(warp);
    }
    auto pieces_of = [&](int units) {
      return units ? max(min((int)(units * (rate * pairs)), a.max_pieces * pairs), pairs) : 0;
    };
    if (aligned) {
      int n = 0;
#pragma unroll 1
      for (int e = lane; e < a.n_tiles; e += 32) n += pieces_of(units_of[e]);
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) sums[warp] = n, rates[warp] = rate;
      __syncthreads();
      const unsigned fits = __ballot_sync(0xffffffffu, lane < WARPS && sums[lane < WARPS ? lane : 0] <= warps);
      aligned = fits != 0;
      if (aligned) rate = rates[__ffs(fits) - 1];
    }
    if (warp == 0) {
      int before = 0;
#pragma unroll 1
      for (int e0 = 0; e0 < a.n_tiles; e0 += 32) {
        const int e = e0 + lane, u = e < a.n_tiles ? units_of[e] : 0;
        const int n = aligned ? pieces_of(u) : u ? (u + KA_BEGIN) * pairs : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += up;
        }
        if (e < a.n_tiles) start[e] = before + incl - n;
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) start[a.n_tiles] = before;
    }
    __syncthreads();
    begin(1);
    if (blockIdx.x == 0)
#pragma unroll 1
      for (int e = tid; e < a.n_tiles; e += 32 * WARPS)
        if (units_of[e] == 0)
          for (int i = 0; i < pairs; ++i) a.desc[e * pairs + i] = make_int4(-1, -1, 0, 0);
    if (total == 0) return;
    me = warp * gridDim.x + blockIdx.x;                       // (few stretches lie on as many SMs)
    x = me, x_end = me + 1;                                   // pieces: one
    if (!aligned) {
      // every head begins with KA_BEGIN places for what that takes
      const int places = start[a.n_tiles], least = max(KA_LONG / 2, (longest + a.max_pieces - 1) / a.max_pieces);
      const int parts = min(max(places / least, 1), warps);
      each = places / parts, longer = places - each * parts;  // the first `longer` have one more
      x = me * each + min(me, longer);
      x_end = me < parts ? x + each + (me < longer ? 1 : 0) : x;
    } else if (me >= start[a.n_tiles]) {
      return;
    }
  }

  const float scale_log2 = a.scale * 1.44269504088896341f;
  const float score_up = scale_log2 * DOWN;
  const int eighths = a.page_size / KV4_EIGHTH;
  unsigned char* my_ring = smem + (size_t)warp * KA_STAGES * UNIT_BYTES;

  while (x < x_end) {
    int e, pair, u0, mine, n_pieces;
    KaTile t;
    KaSpan span;
    if constexpr (HEAD) {
      const int share = AGAIN ? 1 : a.share;
      const int head = AGAIN ? x : blockIdx.x / share, rank = AGAIN ? 0 : blockIdx.x - head * share;
      e = head / pairs, pair = head - e * pairs;
      x = AGAIN ? x + gridDim.x : x_end;
      if constexpr (AGAIN) {
        const int i = e / a.tiles_per_item;
        if (a.beyond[i * a.nkv + pair / a.chunks] == 0 || a.moved[4 * (size_t)i + 2] <= 0) continue;
      }
      t = tile_of(e, !AGAIN && pair == 0 && rank == 0 && tid == 0);
      if (!AGAIN) begin(1);
      if (t.ntok <= 0) {
        if (AGAIN) continue;
        return;
      }
      span = ka_span(t, a.window, a.keep);
      const int steps = (span.units + 1) >> 1, all = WARPS * share, w = warp * share + rank;
      const int few = steps / all, more = steps - few * all;
      u0 = 2 * (w * few + min(w, more));
      mine = max(min(2 * (few + (w < more ? 1 : 0)), span.units - u0), 0), n_pieces = all;
    } else {
      // the tile of x: the last that begins at or before it, among every sixteenth and then among sixteen
      e = lane * 16;
      e = (31 - __clz(__ballot_sync(0xffffffffu, e < a.n_tiles && start[e] <= x))) * 16;
      const int e1 = e + (lane & 15);
      e += 31 - __clz(__ballot_sync(0xffffffffu, lane < 16 && e1 < a.n_tiles && start[e1] <= x));
      static_assert(KA_MAX_TILES <= 512, "two steps");
      t = tiles[e];
      span = ka_span(t, a.window, a.keep);
      const int y = x - start[e];
      if (aligned) {
        const int n = start[e + 1] - start[e], fewer = ka_div(n, pairs), more = n - fewer * pairs;
        const int edge = more * (fewer + 1);                  // the first `more` heads have a piece more
        n_pieces = fewer + (y < edge ? 1 : 0);
        const int z = y < edge ? y : y - edge;
        pair = ka_div(z, n_pieces);
        const int piece = z - pair * n_pieces, units = ka_div(span.units, n_pieces), over = span.units - units * n_pieces;
        if (y >= edge) pair += more;
        u0 = piece * units + min(piece, over);
        mine = units + (piece < over ? 1 : 0);
        x = x_end;
      } else {
        const int v = span.units + KA_BEGIN;
        pair = y / v;
        const int place = y - pair * v, to = min(v, place + x_end - x);
        u0 = max(place - KA_BEGIN, 0);
        mine = to - KA_BEGIN - u0;
        n_pieces = 1;
        if (mine < span.units) {                              // (asked for where u0 is 0: how many warps share the head)
          const int at = x - place + v - 1, edge = longer * (each + 1);
          n_pieces = (at < edge ? at / (each + 1) : longer + (at - edge) / each) - me + 1;
        }
        x += to - place;
        if (mine <= 0) continue;
      }
    }
    const int h = a.chunks == 1 ? pair : pair / a.chunks, head0 = h * a.group + (pair - h * a.chunks) * a.chunk;
    const int heads = min(a.chunk, (h + 1) * a.group - head0);
    const int last = t.pos0 + t.ntok - 1;
    const int* table = a.block_tables + (size_t)t.b * a.table_stride;

    uint4 raw[NT][KW];                                      // the queries, under way while pages are looked up
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + r, ti = n * a.chunk_inverse >> 8, gi = n - ti * a.chunk;
      const bool on = ti < t.ntok && gi < heads;
      const __nv_bfloat16* src =
          a.q + (long long)(t.row0 + (on ? ti : 0)) * a.q_stride + (size_t)(head0 + (on ? gi : 0)) * D;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        raw[nt][w] = *reinterpret_cast<const uint4*>(src + (w >> 1) * 64 + q4 * 16 + (w & 1) * 8);
        if (!on) raw[nt][w] = make_uint4(0, 0, 0, 0);
      }
    }
    // the stretch's units: u0, u0 + 1, ...
    auto unit_key = [&](int i) {
      const int u = u0 + i;
      return (u < span.kept ? u : span.from + u - span.kept) * KA_UNIT;
    };
    int rec0 = 0, rec1 = 0;                                 // of unit (32 n + lane): its two records
    auto record = [&](int j, int n) {                       // of keys j .. j + n - 1, n a page's at most
      if (!kv4_seen(j, j + n - 1, t.pos0, last, a.window, a.keep)) return 0;
      const int at = j >> a.page_shift, page = table[at];
      if (page >= 0 && page < a.num_pages) return (page * a.nkv + h) * eighths + ((j - (at << a.page_shift)) >> 3);
      atomicOr(a.err, BF_ERR_PAGE);
      return 0;
    };
    auto look_up = [&](int i) {
      rec0 = rec1 = 0;
      if (i >= mine) return;
      if (eighths > 1) {
        rec0 = record(unit_key(i), KA_UNIT);
      } else {
        rec0 = record(unit_key(i), 8);
        rec1 = record(unit_key(i) + 8, 8);
      }
    };
    auto issue = [&](int i) {
      if (i >= mine) return;
      unsigned char* dst = my_ring + (i % KA_STAGES) * UNIT_BYTES + lane * 16;
      const unsigned char* s0 = a.cache + (size_t)__shfl_sync(0xffffffffu, rec0, i & 31) * REC + lane * 16;
      if (eighths > 1) {
#pragma unroll
        for (int c0 = 0; c0 < UNIT_BYTES / 16; c0 += 32)
          if (c0 + 32 <= UNIT_BYTES / 16 || c0 + lane < UNIT_BYTES / 16) cp_async16(dst + c0 * 16, s0 + c0 * 16, 16);
      } else {                                              // the second record lies in another page
        const unsigned char* s1 = a.cache + (size_t)__shfl_sync(0xffffffffu, rec1, i & 31) * REC - REC + lane * 16;
#pragma unroll
        for (int c0 = 0; c0 < UNIT_BYTES / 16; c0 += 32)
          if (c0 + 32 <= UNIT_BYTES / 16 || c0 + lane < UNIT_BYTES / 16)
            cp_async16(dst + c0 * 16, (c0 + lane < REC / 16 ? s0 : s1) + c0 * 16, 16);
      }
    };
    auto issue_step = [&](int i) {
      if ((i & 31) == 0) look_up(i + lane);
      issue(i);
      issue(i + 1);
      cp_async_commit();
    };
    issue_step(0);
    issue_step(2);

    // ---- queries: operand b of the scores' product, and their sums per group
    unsigned qf[NT][KW][4], ql[NT][2];
    int pcol[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float qsum[NG] = {};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const unsigned* u = &raw[nt][w].x;
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = __uint_as_float(u[i] << 16);
          f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) qsum[w >> 1] += f[i];
        qf[nt][w][0] = pack_bf16(f[0] * UP, f[4] * UP);
        qf[nt][w][1] = pack_bf16(f[1] * (UP / 16), f[5] * (UP / 16));
        qf[nt][w][2] = pack_bf16(f[2] * UP, f[6] * UP);
        qf[nt][w][3] = pack_bf16(f[3] * (UP / 16), f[7] * (UP / 16));
      }
      // the sums meet the keys' lowest values in one product: lane q4's share is their q4-th bfloat16 term
      float term[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float v = qsum[g];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        v *= scale_log2;
        const float t0 = __bfloat162float(__float2bfloat16_rn(v)), v1 = v - t0;
        const float t1 = __bfloat162float(__float2bfloat16_rn(v1)), v2 = v1 - t1;
        term[g] = q4 == 0 ? t0 : q4 == 1 ? t1 : q4 == 2 ? v2 : 0.f;
      }
      ql[nt][0] = pack_bf16(term[0], term[1]);
      ql[nt][1] = pack_bf16(term[2], term[3]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n2 = nt * 8 + 2 * q4 + i, t2 = n2 * a.chunk_inverse >> 8;
        pcol[nt][i] = t.pos0 + min(t2, t.ntok - 1);
      }
    }

    // p = 2^(s - m), m some 64 below the largest score so far: the probabilities carry their 2^64 from here
    float o[NT][D / 16][4], ps[NT][NG][4], corr[NT][NG][2], l[NT][2], m[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        ps[nt][g][0] = ps[nt][g][1] = ps[nt][g][2] = ps[nt][g][3] = 0.f;
        corr[nt][g][0] = corr[nt][g][1] = 0.f;
      }
      l[nt][0] = l[nt][1] = 0.f;
      m[nt][0] = m[nt][1] = -1e30f;
    }

    // scores of keys r and 8 + r of a unit against columns 2 q4, 2 q4 + 1 of every eight
    auto scores = [&](float (&s)[NT][4], const unsigned char* s0) {
      const unsigned char* s1 = s0 + REC;
      unsigned w0[KW], w1[KW], p0[NG], p1[NG];
      kv4_words<KW>(w0, s0 + r * (D / 2) + q4 * (D / 8));
      kv4_words<KW>(w1, s1 + r * (D / 2) + q4 * (D / 8));
      kv4_words<NG>(p0, s0 + kv4_key_params_at(D) + r * NG * 4);
      kv4_words<NG>(p1, s1 + kv4_key_params_at(D) + r * NG * 4);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int w = 2 * g + half;
          const unsigned a0[4] = {w0[w] & M0, w1[w] & M0, w0[w] & M4, w1[w] & M4};
          const unsigned h0 = w0[w] >> 8, h1 = w1[w] >> 8;
          const unsigned a1[4] = {h0 & M0, h1 & M0, h0 & M4, h1 & M4};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16_16816(c[nt], a0, qf[nt][w][0], qf[nt][w][1]);
            mma_bf16_16816(c[nt], a1, qf[nt][w][2], qf[nt][w][3]);
          }
        }
        const float sc0 = kv4_scale(p0[g]), sc1 = kv4_scale(p1[g]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[nt][0] = fmaf(sc0, c[nt][0], s[nt][0]);
          s[nt][1] = fmaf(sc0, c[nt][1], s[nt][1]);
          s[nt][2] = fmaf(sc1, c[nt][2], s[nt][2]);
          s[nt][3] = fmaf(sc1, c[nt][3], s[nt][3]);
        }
      }
      unsigned low[4] = {0u, 0u, 0u, 0u};                   // (m of group 0, m of group 1), of 2 and 3
      low[0] = NG > 1 ? __byte_perm(p0[0], p0[NG > 1 ? 1 : 0], 0x7632) : p0[0] >> 16;
      low[1] = NG > 1 ? __byte_perm(p1[0], p1[NG > 1 ? 1 : 0], 0x7632) : p1[0] >> 16;
      if (NG > 2) {
        low[2] = __byte_perm(p0[NG > 2 ? 2 : 0], p0[NG > 2 ? 3 : 0], 0x7632);
        low[3] = __byte_perm(p1[NG > 2 ? 2 : 0], p1[NG > 2 ? 3 : 0], 0x7632);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        mma_bf16_16816(c, low, ql[nt][0], ql[nt][1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[nt][k] = fmaf(s[nt][k], score_up, c[k]);
      }
    };
    // adds a unit's values; `hidden`: bits of elements whose key the column does not see
    auto values = [&](float (&s)[NT][4], const unsigned char* s0, auto edge, unsigned hidden) {
      const unsigned char* s1 = s0 + REC;
      unsigned v0[KW], v1[KW], p0[NG], p1[NG];
      kv4_words<KW>(v0, s0 + kv4_values_at(D) + r * (D / 2) + q4 * (D / 8));
      kv4_words<KW>(v1, s1 + kv4_values_at(D) + r * (D / 2) + q4 * (D / 8));
      kv4_words<NG>(p0, s0 + kv4_value_params_at(D) + r * NG * 4);
      kv4_words<NG>(p1, s1 + kv4_value_params_at(D) + r * NG * 4);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int k = 0; k < 4; ++k) s[nt][k] = ka_exp2(s[nt][k] - m[nt][k & 1]);
        l[nt][0] += s[nt][0] + s[nt][2];
        l[nt][1] += s[nt][1] + s[nt][3];
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float sc0 = kv4_scale(p0[g]), sc1 = kv4_scale(p1[g]);
        const float mid0 = fmaf(8.f, sc0, kv4_low(p0[g])), mid1 = fmaf(8.f, sc1, kv4_low(p1[g]));
        unsigned b0[NT], b1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4] = {s[nt][0] * sc0, s[nt][1] * sc0, s[nt][2] * sc1, s[nt][3] * sc1};
          if constexpr (decltype(edge)::value) {            // (a hidden key may be anything: 0 times it is not 0)
            float z[4] = {s[nt][0] * mid0, s[nt][1] * mid0, s[nt][2] * mid1, s[nt][3] * mid1};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (hidden >> (nt * 4 + k) & 1) w[k] = z[k] = 0.f;
            corr[nt][g][0] += z[0] + z[2];
            corr[nt][g][1] += z[1] + z[3];
          } else {
            corr[nt][g][0] = fmaf(s[nt][2], mid1, fmaf(s[nt][0], mid0, corr[nt][g][0]));
            corr[nt][g][1] = fmaf(s[nt][3], mid1, fmaf(s[nt][1], mid0, corr[nt][g][1]));
          }
          b0[nt] = ka_transpose(pack_bf16(w[0], w[1]));
          b1[nt] = ka_transpose(pack_bf16(w[2], w[3]));
          const unsigned ones[4] = {ONES, ONES, ONES, ONES};
          mma_bf16_16816(ps[nt][g], ones, b0[nt], b1[nt]);
        }
        // eight numbers of this lane's part, for tokens 2 q4 and 2 q4 + 1 of either record
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned sel = half ? 0x7632 : 0x5410;
          const unsigned x0 = __byte_perm(v0[g], v0[NG + g], sel), x1 = __byte_perm(v1[g], v1[NG + g], sel);
          const unsigned y0 = x0 & M8, y1 = x1 & M8, z0 = __byte_perm(x0, 0u, 0x4341), z1 = __byte_perm(x1, 0u, 0x4341);
          const unsigned a0[4] = {y0 & M0, y0, y1 & M0, y1};
          const unsigned a1[4] = {z0 & M0, z0, z1 & M0, z1};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_bf16_16816(o[nt][4 * g + 2 * half], a0, b0[nt], b1[nt]);
            mma_bf16_16816(o[nt][4 * g + 2 * half + 1], a1, b0[nt], b1[nt]);
          }
        }
      }
    };
    // two units at a time, so that one's latencies lie under the other's work
    auto step = [&](int i, auto edge) {
      const unsigned char* sa = my_ring + (i % KA_STAGES) * UNIT_BYTES;
      const unsigned char* sb = sa + UNIT_BYTES;
      float s[2][NT][4];
      scores(s[0], sa);
      scores(s[1], sb);
      unsigned hidden[2] = {0u, 0u};
      if constexpr (decltype(edge)::value) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = i + u < mine ? unit_key(i + u) : 0x7fffff00;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = key + r + (k >> 1) * 8, p = pcol[nt][k & 1];
              if (j > p || (a.window > 0 && j <= p - a.window && j >= a.keep)) {
                hidden[u] |= 1u << (nt * 4 + k);
                s[u][nt][k] = -INFINITY;
              }
            }
        }
      }
      bool over = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[nt][c] = fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2]));
          over |= top[nt][c] > m[nt][c] + 72.f;
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = top[nt][c];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x - 64.f, m[nt][c]);
            const float f = ka_exp2(m[nt][c] - x);
            m[nt][c] = x;
            l[nt][c] *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              corr[nt][g][c] *= f;
              ps[nt][g][c] *= f;
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[nt][d][c] *= f;
              o[nt][d][c + 2] *= f;
            }
          }
      }
      values(s[0], sa, edge, hidden[0]);
      values(s[1], sb, edge, hidden[1]);
    };
    // units whose every key every column sees: not so at the context's end and at the window's edges
    const int inner = span.kept - u0;                       // (units of kept tokens count as edges)
    const int from_i = a.window > 0 ? inner + max(0, (max(0, last - a.window + 1) + KA_UNIT - 1) / KA_UNIT - span.from) : 0;
    const int to_i = min(mine, inner + (t.pos0 + 1) / KA_UNIT - span.from);
    for (int i = 0; i < mine; i += 2) {
      cp_async_wait<1>();
      __syncwarp();
      if (i >= from_i && i + 2 <= to_i) step(i, Bool<false>()); else step(i, Bool<true>());
      __syncwarp();
      issue_step(i + 4);
    }
    cp_async_wait<0>();

    // ---- the result: lane (r, q4) has numbers 8 r .. 8 r + 7 of every group, of two columns of every eight
    const bool whole = !HEAD && mine == span.units;
    const int slot = HEAD ? warp : 2 * me + (u0 == 0 ? 1 : 0);
    // (HEAD: over the ring; eight numbers between rows, so that stores meet in two ways only)
    constexpr int ROW = HEAD ? D + 8 : D;
    float* part_o = HEAD ? reinterpret_cast<float*>(smem) : a.part_o;
    float2* part_ml = HEAD ? reinterpret_cast<float2*>(tiles) : a.part_ml;
    static_assert(!HEAD || (COLS * ROW * 4 <= KA_STAGES * UNIT_BYTES && WARPS * COLS * 8 <= KA_MAX_TILES * 16), "room");
    if (HEAD) __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = nt * 8 + 2 * q4 + c, ti = n * a.chunk_inverse >> 8, gi = n - ti * a.chunk;
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], k);
#pragma unroll
          for (int g = 0; g < NG; ++g) corr[nt][g][c] += __shfl_xor_sync(0xffffffffu, corr[nt][g][c], k);
        }
        if (ti >= t.ntok || gi >= heads) continue;
        const float sum = l[nt][c] * (1.f / UP);
        const float f = whole ? 1.f / sum : 1.f;
        if (!whole && r == 0) part_ml[slot * COLS + n] = make_float2(m[nt][c], sum);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float base = fmaf(-8.f * DOWN, ps[nt][g][c], corr[nt][g][c] * (1.f / UP));
          float v[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[2 * k] = fmaf(o[nt][4 * g + k][c], DOWN, base) * f;
            v[2 * k + 1] = fmaf(o[nt][4 * g + k][c + 2] - o[nt][4 * g + k][c], DOWN / 16, base) * f;
          }
          if (whole) {
            *reinterpret_cast<uint4*>(a.out + (long long)(t.row0 + ti) * a.out_stride + (size_t)(head0 + gi) * D + g * 64 + r * 8) =
                make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
          } else {
            float4* dst = reinterpret_cast<float4*>(part_o + ((size_t)slot * COLS + n) * ROW + g * 64 + r * 8);
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
    if constexpr (HEAD) {
      // a column by one warp, or two warps, a warp one or two columns
      constexpr int PER = WARPS > COLS ? WARPS / COLS : 1, N = D / PER / 32, IDS = COLS * PER / WARPS;
      static_assert(COLS * PER % WARPS == 0, "columns");
      __syncthreads();
      float acc[IDS][N], sum[IDS], top[IDS];
      auto on = [&](int n) {
        const int ti = n * a.chunk_inverse >> 8;
        return ti < t.ntok && n - ti * a.chunk < heads;
      };
      auto finish = [&](int id, const float (&v)[N], float l) {
        const int n = id / PER, ti = n * a.chunk_inverse >> 8, gi = n - ti * a.chunk;
        __nv_bfloat16* dst = a.out + (long long)(t.row0 + ti) * a.out_stride + (size_t)(head0 + gi) * D +
                             id % PER * (D / PER);
#pragma unroll
        for (int k = 0; k < N; ++k) dst[lane + 32 * k] = __float2bfloat16_rn(v[k] / l);
      };
#pragma unroll
      for (int j = 0; j < IDS; ++j) {
        const int id = warp + j * WARPS, n = id / PER;
        if (!on(n)) continue;
        const float2 ml = lane < WARPS ? part_ml[lane * COLS + n] : make_float2(-INFINITY, 0.f);
        top[j] = ml.x;
#pragma unroll
        for (int k = 1; k < WARPS; k <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], k));
        const float f = ml.x == top[j] ? 1.f : ka_exp2(ml.x - top[j]);
        sum[j] = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) acc[j][k] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float g = __shfl_sync(0xffffffffu, f, w);
          sum[j] = fmaf(g, __shfl_sync(0xffffffffu, ml.y, w), sum[j]);
#pragma unroll
          for (int k = 0; k < N; ++k)
            acc[j][k] = fmaf(g, part_o[(w * COLS + n) * ROW + id % PER * (D / PER) + lane + 32 * k], acc[j][k]);
        }
        if (AGAIN || a.share == 1) finish(id, acc[j], sum[j]);
      }
      if constexpr (AGAIN) __syncthreads();                 // (the next head's ring lies over the partials)
      if (!AGAIN && a.share > 1) {
        // the blocks' sums, a column by one warp of one of them
        const int rank = blockIdx.x % a.share;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < IDS; ++j) {
          const int id = warp + j * WARPS, n = id / PER;
          if (!on(n)) continue;
#pragma unroll
          for (int k = 0; k < N; ++k) part_o[n * D + id % PER * (D / PER) + lane + 32 * k] = acc[j][k];
          if (id % PER == 0 && lane == 0) part_ml[n] = make_float2(top[j], sum[j]);
        }
        ka_cluster_sync();
#pragma unroll 1
        for (int id = warp * a.share + rank; id < COLS * PER; id += WARPS * a.share) {
          const int n = id / PER;
          if (!on(n)) continue;
          float m1 = -INFINITY, l1 = 0.f;
          if (lane < a.share) m1 = ka_peer(&part_ml[n].x, lane), l1 = ka_peer(&part_ml[n].y, lane);
          float part[KA_SHARE][N];
#pragma unroll
          for (int c = 0; c < KA_SHARE; ++c)
#pragma unroll
            for (int k = 0; k < N; ++k)
              part[c][k] = c < a.share ? ka_peer(part_o + n * D + id % PER * (D / PER) + lane + 32 * k, c) : 0.f;
          float most = m1;
#pragma unroll
          for (int k = 1; k < KA_SHARE; k <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k));
          const float f = m1 == most ? 1.f : ka_exp2(m1 - most);
          float l = 0.f, v[N];
#pragma unroll
          for (int k = 0; k < N; ++k) v[k] = 0.f;
#pragma unroll
          for (int c = 0; c < KA_SHARE; ++c) {
            const float g = __shfl_sync(0xffffffffu, f, c);
            l = fmaf(g, __shfl_sync(0xffffffffu, l1, c), l);
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = fmaf(g, part[c][k], v[k]);
          }
          finish(id, v, l);
        }
        ka_cluster_sync();                                  // (this block's memory may be read until here)
      }
    } else if (u0 == 0 && lane == 0)
      a.desc[e * pairs + pair] = whole ? make_int4(-1, -1, 0, 0) : make_int4(me, n_pieces, t.row0, t.ntok);
  }
}

// Adds up what several warps left of a (tile, head).  A block of eight warps has 8 / PER columns, PER warps
// take a column's partials in turn (one where a head has few of them).  Partials and their maxima are
// asked for together; warps meet in shared memory.
template <int D, int PER>
__global__ void __launch_bounds__(256)
kv4_merge_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                 const int4* __restrict__ desc, __nv_bfloat16* __restrict__ out, long long out_stride, int group,
                 int chunk, int chunks, unsigned chunk_inverse, int pairs, int cols) {
  constexpr int N = D / 32, DEPTH = D == 256 ? 4 : 8;
  __shared__ float sh_o[PER > 1 ? 8 : 1][D], sh_m[8], sh_l[8];
  bf_pdl_trigger();
  bf_pdl_wait();
  const int4 d = desc[blockIdx.x];
  if (d.x < 0) return;
  const int pair = blockIdx.x % pairs, h = pair / chunks, head0 = h * group + (pair - h * chunks) * chunk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = blockIdx.y * (8 / PER) + warp / PER, ti = n * chunk_inverse >> 8, gi = n - ti * chunk;
  if (ti >= d.w || gi >= min(chunk, (h + 1) * group - head0)) return;    // (PER > 1: the whole block)
  float top = -INFINITY, sum = 0.f, acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  for (int i0 = warp % PER; i0 < d.y; i0 += PER * DEPTH) {
    float2 ml[DEPTH];
    float v[DEPTH][N];
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      const int i = i0 + j * PER;
      ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < N; ++k) v[j][k] = 0.f;
      if (i < d.y) {
        const size_t slot = (size_t)(2 * (d.x + i) + (i == 0 ? 1 : 0)) * cols + n;
        ml[j] = part_ml[slot];
#pragma unroll
        for (int k = 0; k < N; ++k) v[j][k] = part_o[slot * D + lane + 32 * k];
      }
    }
    float next = top;
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) next = fmaxf(next, ml[j].x);
    const float f = ka_exp2(top - next);                    // (the first time 0 times 0)
    sum *= f;
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] *= f;
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      const float g = ml[j].x == next ? 1.f : ka_exp2(ml[j].x - next);
      sum = fmaf(g, ml[j].y, sum);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = fmaf(g, v[j][k], acc[k]);
    }
    top = next;
  }
  __nv_bfloat16* dst = out + (long long)(d.z + ti) * out_stride + (size_t)(head0 + gi) * D;
  if (PER == 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) dst[lane + 32 * k] = __float2bfloat16_rn(acc[k] / sum);
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) sh_o[warp][lane + 32 * k] = acc[k];
  if (lane == 0) sh_m[warp] = top, sh_l[warp] = sum;
  __syncthreads();
  if (threadIdx.x < D) {
    float most = sh_m[0], v = 0.f, w = 0.f;
#pragma unroll
    for (int k = 1; k < 8; ++k) most = fmaxf(most, sh_m[k]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = sh_m[k] == most ? 1.f : ka_exp2(sh_m[k] - most);
      v = fmaf(f, sh_o[k][threadIdx.x], v);
      w = fmaf(f, sh_l[k], w);
    }
    dst[threadIdx.x] = __float2bfloat16_rn(v / w);
  }
}

template <int D, int NT>
static int ka_launch(KaArgs a, int total_tiles, int share, int sms, cudaStream_t stream) {
  constexpr int threads = 32 * ka_warps(D, NT);
  constexpr size_t smem = (size_t)ka_warps(D, NT) * KA_STAGES * 2 * kv4_record(D) +
                          KA_MAX_TILES * (sizeof(KaTile) + 4) + (KA_MAX_TILES + 4) * 4;
  static bool configured[BF_MAX_DEVICES];
  const int dev = bf_current_device();
  if (!configured[dev]) {
    for (auto kern : {kv4_attention_kernel<D, NT, KA_STRETCHES>, kv4_attention_kernel<D, NT, KA_HEAD>,
                      kv4_attention_kernel<D, NT, KA_AGAIN>}) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return (int)e;
    }
    configured[dev] = true;
  }
  const int pairs = a.nkv * a.chunks;
  if (a.beyond) {
    const long long heads = (long long)total_tiles * pairs;
    if (heads > 0x7fffffffLL - sms) return (int)cudaErrorInvalidValue;
    a.heads = (int)heads;
    return bf_launch_pdl(kv4_attention_kernel<D, NT, KA_AGAIN>, dim3(heads < sms ? (int)heads : sms), dim3(threads),
                         smem, stream, a);
  }
  // the units of a launch are counted in 32 bits
  const long long units = ((long long)a.table_width * a.page_size / KA_UNIT + 2 + KA_BEGIN) * pairs;
  if (units > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const int most = 0x7fffffffLL / units < KA_MAX_TILES ? (int)(0x7fffffffLL / units) : KA_MAX_TILES;
  if (share) {
    a.share = share;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(total_tiles * pairs * share);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = bf_pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = share, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_attention_kernel<D, NT, KA_HEAD>, a);
    return e != cudaSuccess ? (int)e : bf_launch_status();
  }
  for (int first = 0; first < total_tiles; first += most) {
    a.first_tile = first;
    a.n_tiles = total_tiles - first < most ? total_tiles - first : most;
    // heads with many pieces each (there are few of them): eight warps add a column's up
    const bool few = (long long)a.n_tiles * pairs * 8 < (long long)sms * ka_warps(D, NT);
    a.max_pieces = few ? sms * ka_warps(D, NT) : 64;
    int e = bf_launch_pdl(kv4_attention_kernel<D, NT, KA_STRETCHES>, dim3(sms), dim3(threads), smem, stream, a);
    if (e) return e;
    auto merge = [&](auto kern, int columns) {
      return bf_launch_pdl(kern, dim3(a.n_tiles * pairs, 8 * NT / columns), dim3(256), 0, stream,
                           (const float*)a.part_o, (const float2*)a.part_ml, (const int4*)a.desc, a.out,
                           a.out_stride, a.group, a.chunk, a.chunks, a.chunk_inverse, pairs, 8 * NT);
    };
    e = few ? merge(kv4_merge_kernel<D, 8>, 1) : merge(kv4_merge_kernel<D, 1>, 8);
    if (e) return e;
  }
  return 0;
}

// Columns of a tile for `group` query heads per kv head: heads of a chunk, chunks, token rows.
struct KaShape {
  int nt, chunk, chunks, tokens;
};
static KaShape ka_shape(int group, int d, int max_rows) {
  // Two sets of eight columns where one would leave heads out or a portion's rows come one by one; heads
  // of 256 have no registers for a second one.
  KaShape s;
  s.nt = d <= 128 && (group > 8 || max_rows > 8 / (group < 8 ? group : 8)) ? 2 : 1;
  const int cols = 8 * s.nt;
  s.chunks = (group + cols - 1) / cols;
  s.chunk = (group + s.chunks - 1) / s.chunks;
  s.tokens = cols / s.chunk < max_rows ? cols / s.chunk : max_rows;
  return s;
}

static long long ka_slots(const KaShape& s, int d, int sms) { return 2LL * sms * ka_warps(d, s.nt); }

// Blocks that each (tile, head) gets for itself, as a cluster whose warps meet in shared memory; 0: stretches of
// equal work and a second kernel.  `keys`: the most that a tile can see.  The faster by what both take, in us, from a
// sweep of rows of equal length (replayed from a graph, launch included): a cluster 6.5 (several blocks 8.5) and `unit`
// for each unit of a block, where all clusters are resident at once (74, 33 and 15 of two, four and eight blocks);
// stretches `base`, `each` for every unit of all heads, of which a batch has three quarters of what its longest row
// says (all of it where a window cuts them to one length, `even`), and `piece` for a head's pieces.  Heads of 128
// (4 query heads each), stretches / 1, 2, 4, 8 blocks: 8 heads over 512 keys 10.7 / 8.6, 8.6, 8.6, 8.6, over 4,096
// 12.6 / 20.9, 14.8, 12.7, 10.6, over 16,384 19.0 / 62, 36, 23, 15.4; 32 heads over
// 4,096 16.9 / 20.9, 14.7, 12.7; 72 over 4,096 19.0 / 20.9, 16.3; 128 over 512 14.7 / 8.7, over 4,096 27.2 / 21.0.
static int ka_blocks_a_head(const KaShape& s, int d, long long tiles, int pairs, int keys, bool even, int sms) {
  struct Times {
    float unit, base, each, piece;
  };
  const Times t = d == 64    ? (s.nt == 1 ? Times{0.033f, 9.2f, 0.5e-3f, 0.011f} : Times{0.05f, 9.5f, 0.8e-3f, 0.011f})
                  : d == 128 ? (s.nt == 1 ? Times{0.056f, 11.5f, 0.45e-3f, 0.011f} : Times{0.094f, 11.5f, 1.0e-3f, 0.011f})
                             : Times{0.105f, 12.f, 0.7e-3f, 0.035f};
  const float units = keys / KA_UNIT + 1, heads = (float)tiles * pairs;
  const float pieces = fminf(sqrtf(KA_PIECES * units), sms * ka_warps(d, s.nt) / heads);
  float best = t.base + t.each * units * heads * (tiles > 1 && !even ? 0.75f : 1.f) + t.piece * pieces;
  int share = 0;
  for (int c = 1; c <= KA_SHARE; c *= 2) {
    const int fit = sms * (c < 4 ? 100 : c == 4 ? 90 : 82) / (100 * c);
    const float time = (c == 1 ? 6.5f : 8.5f) + t.unit * units / c;
    if (heads <= fit && time < best) best = time, share = c;
  }
  return share;
}

// Bytes of scratch that a call needs (16-byte aligned): partial results and a note per (tile, head); none where
// no second kernel runs.  `keys`, `even` as the call's.
BF_EXPORT long long bf_kv4_attention_scratch(int n, int max_rows, int nh, int nkv, int d, int sms, int keys, int even) {
  const KaShape s = ka_shape(nh / nkv, d, max_rows);
  const long long all = (long long)n * ((max_rows + s.tokens - 1) / s.tokens);
  if (ka_blocks_a_head(s, d, all, nkv * s.chunks, keys, even, sms)) return 0;
  const long long slots = ka_slots(s, d, sms);
  long long tiles = (long long)n * ((max_rows + s.tokens - 1) / s.tokens);
  if (tiles > KA_MAX_TILES) tiles = KA_MAX_TILES;
  return slots * 8 * s.nt * (d * 4 + 8) + tiles * nkv * s.chunks * 16;
}

struct Kv4AttentionCall {
  const void* q;
  long long q_stride;
  const void* cache;
  const int* rows, *seq_of_token, *positions, *items;
  int n, max_rows, T;
  const int* block_tables;
  int table_stride, table_rows, table_width;
  void* out;
  long long out_stride;
  int nh, nkv, d, page_size, num_pages, window, keep;
  float scale;
  void* scratch;
  int sms, keys, even;                                     // what a row can see, as to the scratch
  int early;                                               // the description was there before the kernel ahead began
  int* err;
  cudaStream_t stream;
  // or null: only the portions and kv heads that `beyond` [n, nkv] notes, where `moved` [n, 4] has rows for them (no
  // scratch)
  const int *beyond, *moved;
};
BF_EXPORT int bf_kv4_attention(const Kv4AttentionCall* call) {
  const auto& [q, q_stride, cache, rows, seq_of_token, positions, items, n, max_rows, T, block_tables,
               table_stride, table_rows, table_width, out, out_stride, nh, nkv, d, page_size, num_pages,
               window, keep, scale, scratch, sms, keys, even, early, err, stream, beyond, moved] = *call;
  if (n <= 0 || max_rows <= 0) return 0;
  if ((long long)num_pages * nkv * (page_size / 8) > 0x7fffffffLL || page_size < 8 || (page_size & (page_size - 1)) ||
      (long long)table_width * page_size > 1 << 24)        // (a tile's units stay below 2^20)
    return (int)cudaErrorInvalidValue;
  const KaShape s = ka_shape(nh / nkv, d, max_rows);
  KaArgs a = {};
  a.q = (const __nv_bfloat16*)q, a.q_stride = q_stride, a.cache = (const unsigned char*)cache;
  a.rows = rows, a.seq_of_token = seq_of_token, a.positions = positions, a.items = items;
  a.tiles_per_item = (max_rows + s.tokens - 1) / s.tokens;
  a.T = T, a.block_tables = block_tables;
  a.table_stride = table_stride, a.table_rows = table_rows, a.table_width = table_width;
  a.out = (__nv_bfloat16*)out, a.out_stride = out_stride;
  a.nh = nh, a.nkv = nkv, a.group = nh / nkv, a.chunk = s.chunk, a.chunks = s.chunks, a.tokens = s.tokens;
  a.page_size = page_size, a.page_shift = 3;
  while (1 << a.page_shift < page_size) ++a.page_shift;
  a.num_pages = num_pages, a.window = window, a.keep = keep, a.scale = scale;
  a.early = early != 0 && !beyond;
  a.beyond = beyond, a.moved = moved, a.n_items = n;
  a.chunk_inverse = (256 + s.chunk - 1) / s.chunk;
  const long long slots = ka_slots(s, d, sms);
  a.part_o = (float*)scratch;
  a.part_ml = (float2*)(a.part_o + slots * 8 * s.nt * d);
  a.desc = (int4*)(a.part_ml + slots * 8 * s.nt);
  a.err = err;
  const long long tiles = (long long)n * a.tiles_per_item;
  if (tiles > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  if (beyond && (!items || !moved)) return (int)cudaErrorInvalidValue;
  const int share = beyond ? 1 : ka_blocks_a_head(s, d, tiles, nkv * s.chunks, keys, even, sms);
  if (!share && !scratch) return (int)cudaErrorInvalidValue;
  if (d == 64)
    return s.nt == 1 ? ka_launch<64, 1>(a, (int)tiles, share, sms, stream)
                     : ka_launch<64, 2>(a, (int)tiles, share, sms, stream);
  if (d == 128)
    return s.nt == 1 ? ka_launch<128, 1>(a, (int)tiles, share, sms, stream)
                     : ka_launch<128, 2>(a, (int)tiles, share, sms, stream);
  if (d == 256) return ka_launch<256, 1>(a, (int)tiles, share, sms, stream);
  return (int)cudaErrorInvalidValue;
}
