// Causal attention with grouped heads on the 5th-generation tensor cores, for
// whole packed prompts and for chunks of new tokens over a paged cache.
//
// A tile's 128 query rows are the `group` query heads that share one key /
// value head, for tpt = 128 / group consecutive tokens (row = token * group +
// head), so K and V are read once for the whole group, a chunk of few
// tokens still fills a tile, and the triangle wastes little: only blocks that
// some row of the tile sees are visited.
//
// Work unit: (request, key/value head, 2 * tpt tokens[, part of the keys]): two
// tiles, whose softmax and MMAs overlap. A unit of one tile (a short chunk, or
// all units where there are few) gives both softmax groups the same rows, each
// with half of the keys; tile 0's group joins the two at the end.
// Requests' offsets are device data, so each CTA finds its units itself.
//  * Prompts: units are numbered without knowing the offsets. Request i
//    starts at virtual tile cu[i] / tu + i, which leaves room for its tiles
//    and at most one empty one behind them, and is found by searching cu. Units
//    are handed out last tokens first (the longest rows first), by cluster
//    launch control: a CTA takes over units whose CTAs have not started, so no
//    counter in memory is needed. It asks when the last loads of its unit are
//    under way and no sooner: a unit held early is one that an idle CTA lacks.
//    The search needs ascending offsets. Where some are not, it may miss sequences
//    that are in order themselves, and warp 11 hands all their units out again.
//  * Paged chunks: few units of very different lengths, so all units' keys
//    (and kUnitKeys more for each unit's ends) are laid end to end and cut into one
//    range per CTA. A unit that a cut falls into leaves parts in the
//    workspace, joined by a second launch; cuts near a unit's ends move there.
//
// CTA: 384 threads, as the non-causal kernel divides them:
//   warps 0-3 / 4-7  softmax of tile 0 / 1, one query row per thread
//   warp 8           TMA producer: Q, then K_j, V_j into an NST-slot ring
//   warp 9           MMA issuer and TMEM owner
//   warp 10          scheduler: finds the units, one ahead
//   warp 11          prompts: looks through all sequences for bad offsets, and
//                    goes on for the scheduler behind its last unit
// MMA order per key block j: PV0_j, S0_{j+1}, PV1_j, S1_{j+1}, each tile with
// its own number of blocks. The first blocks need no mask; in those that reach
// past a row's last key the scores are set to -inf (so P is exactly 0), P V
// stops at the last key rounded up to 16, and the V rows in between are
// zeroed in shared memory: what lies behind a request's keys may be NaN.
//
// Bound by the tensor pipe at the rate of M = 128, N = 128 instructions (about
// 68 % of dense) where there are many blocks. Device time of ten calls in a row:
// 8192 tokens, 32 / 8 heads of 128, 434 us = 1268 TFLOP/s of the causal flops;
// heads of 64 363 us (P V of N = 64 costs what N = 128 does); 6 chunks of 300 -
// 700 tokens behind 2k - 12k keys 258 us. Many more calls in a row run under the
// power cap (the 8192 tokens then take 508 us, the chunks 307). The issuing lane
// must not add to that: with a descriptor built and a lane elected per
// instruction the 8192 tokens took 8 % longer, with heads of 64 12 %. Where there
// are few blocks, bound by its start and the unit boundary (77 tokens: 8.0 us).
//
// Scores and softmax state are fp32, P is rounded to the inputs' type (half
// a step, the rounding V's own type has; fp32 P would need a tf32 product at
// a quarter of the rate), and the row sum takes P before that rounding.
#pragma once
#include "fa_tc.cuh"
#include "paged_rows.cuh"

namespace llmr {

constexpr int kUnitSlots = 2;  // the unit in work and the next
constexpr int kMaxRanges = 160;  // CTAs of a paged call (workspace)
// What a unit costs besides its keys, in keys (24 x 5 drafted tokens: 256 38.0 us,
// 128 39.2, 512 39.1; 200 tokens over 1500 keys 28.5, 28.3, 29.8);
// blocks of 128 that a cut keeps away from a unit's ends (a part costs about
// two blocks to write and join; 6 took the 200 tokens from 28.5 to 37.6 us and
// the drafted ones from 38.0 to 41.2); least keys of a range (with 1024, 20 tokens
// over 100 keys, 8 small units, ran on two SMs: 20.7 us instead of 12.7).
constexpr int kUnitKeys = 256;
constexpr int kCutBlocks = 3;
constexpr int kRangeKeys = 256;
// Prompts with a bad offset: the most CTAs that all units are dealt out to.
constexpr int kMaxShares = 256;

// A unit that a cut falls into, entered by the CTA that begins it: its parts
// are that CTA's second part and the first parts of the CTAs up to `last`.
struct FaJoin {
  int last;  // -1: the CTA begins no such unit
  int q_row, tokens, kvh;
};

struct FaRowsParams {
  RowsParams rows;
  int group, tpt, recip;  // recip: r / group = r * recip >> 16 for r < 128
  int tu;                 // tokens per unit: tpt or 2 * tpt
  int vtiles;             // prompts: virtual tiles of all requests
  int units;              // prompts: vtiles * Hk
  int dynamic;            // prompts: units are taken over by cluster launch control
  int shares;             // prompts: CTAs that units are dealt out to if an offset is bad
  float scale_log2;
  float *part_o;    // paged: [2 * CTA + 0 / 1][256 rows][D], relative to the part's maximum
  float2 *part_ml;  // paged: [2 * CTA + 0 / 1][256 rows] (maximum, sum), in powers of 2
  FaJoin *joins;             // paged: [CTA]
};

// One unit, as the scheduler hands it to the other warps.
struct FaUnit {
  int kvh;         // -1: no more units
  int q_row;       // first token's row in q and o
  int tokens;      // tokens of the unit (tile 0 takes the first tpt)
  int kv_row;      // packed: the sequence's first row; paged: the request
  int keys;        // keys the unit's last row sees
  int pos;         // position of the first token
  int blk;         // first key block
  int nb[2];       // key blocks of each tile
  int dual;        // the tiles are the same rows, tile 1 with the blocks behind tile 0's
  int part;        // -1, or where the partial result goes
};

// The request that virtual tile vt belongs to: the last with
// cu[i] / tu + i <= vt. Whole warp, 32 probes at a time.
__device__ __forceinline__ int find_request(const int *cu, int n, int tu, int vt) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const bool le = i < hi && cu[i] / tu + i <= vt;
    const int c = max(1, __popc(__ballot_sync(0xffffffffu, le)));
    lo += (c - 1) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

// Tile `tile` of a request: all of a unit but its range of key blocks.
__device__ __forceinline__ void unit_rows(FaUnit &un, int tu, int kvh, int row0, int nq, int nk, int tile) {
  const int first = tile * tu;
  un.kvh = kvh;
  un.q_row = row0 + first;
  un.tokens = min(tu, nq - first);
  un.pos = nk - nq + first;
  un.keys = max(0, un.pos + un.tokens);
  un.part = -1;
}
// Key blocks [b0, b1) of the unit. Two tiles of tokens see what their last
// token sees; one tile's rows go to both, each with half of the blocks.
__device__ __forceinline__ void unit_blocks(FaUnit &un, int tpt, int b0, int b1) {
  const int k0 = max(0, un.pos + min(un.tokens, tpt));
  un.blk = b0;
  un.dual = un.tokens <= tpt;
  un.nb[0] = un.dual ? (b1 - b0 + 1) / 2 : max(0, min((k0 + 127) / 128, b1) - b0);
  un.nb[1] = un.dual ? (b1 - b0) / 2 : b1 - b0;
}

// Prompts: virtual unit u; false if it is empty. Whole warp.
__device__ __forceinline__ bool prompt_unit(const FaRowsParams &p, int u, FaUnit &un) {
  const int vt = p.vtiles - 1 - u / p.rows.Hk, tu = p.tu;
  const int r = find_request(p.rows.cu, p.rows.n, tu, vt);
  int row0, nq, nk;
  if (!request_rows(p.rows, r, row0, nq, nk)) return false;
  const int tile = vt - (row0 / tu + r);
  if (tile < 0 || tile >= (nq + tu - 1) / tu) return false;
  unit_rows(un, tu, u % p.rows.Hk, row0, nq, nk, tile);
  un.kv_row = row0;
  unit_blocks(un, p.tpt, 0, (un.keys + 127) / 128);
  return true;
}

// Prompts whose offsets are not all in order: gives each unit of one share of the
// sequences that are, and that begin behind the earlier ones (so a row has one
// sequence). Whole warp; false once give() is.
template <typename Give>
__device__ __forceinline__ bool deal_units(const FaRowsParams &p, int share, Give give) {
  const RowsParams &rp = p.rows;
  const int lane = threadIdx.x & 31, tu = p.tu;
  FaUnit un;
  int end = 0;  // of the sequences so far
  int at = 0;   // their units, modulo p.shares
  for (int r0 = 0; r0 < rp.n; r0 += 32) {
    int row0 = 0, nq = 0, nk = 0;
    if (r0 + lane < rp.n) request_rows(rp, r0 + lane, row0, nq, nk);
    for (unsigned left = __ballot_sync(0xffffffffu, nq > 0); left; left &= left - 1) {
      const int first = __shfl_sync(0xffffffffu, row0, __ffs(left) - 1);
      const int rows = __shfl_sync(0xffffffffu, nq, __ffs(left) - 1);
      if (first < end) continue;
      end = first + rows;
      const long long units = (long long)((rows + tu - 1) / tu) * rp.Hk;
      for (long long x = share < at ? share - at + p.shares : share - at; x < units; x += p.shares) {
        unit_rows(un, tu, (int)(x % rp.Hk), first, rows, rows, (int)(x / rp.Hk));
        un.kv_row = first;
        unit_blocks(un, p.tpt, 0, (un.keys + 127) / 128);
        if (!give(un)) return false;
      }
      at = (int)((at + units) % p.shares);
    }
  }
  return true;
}

// Paged: where tile i of a request begins, in keys from the request's first:
// tile j counts its last token's position (as if it were full) and kUnitKeys.
__host__ __device__ __forceinline__ long long tile_begin(long long ctx, long long tu, long long i) {
  return i * (ctx + kUnitKeys) + tu * (i * (i + 1) / 2);
}
// Paged: the block that a cut `y` keys into a unit of `blocks` blocks falls
// on; a few blocks at either end belong to the neighbour.
__host__ __device__ __forceinline__ int cut_block(long long y, int blocks) {
  const long long b = y <= kUnitKeys ? 0 : (y - kUnitKeys) / 128;
  if (b < kCutBlocks) return 0;
  return b > blocks - kCutBlocks ? blocks : (int)b;
}
// Beginning of range c of `ranges`.
__host__ __device__ __forceinline__ long long cut_at(long long line, int ranges, int c) {
  return line / ranges * c + line % ranges * c / ranges;
}

// A cut of the line: request, head, tile, key block, and where that tile's unit
// begins in the line; r = n behind the last.
struct FaCut {
  int r, kvh, tile, blk;
  long long begin;
};

template <int D>
struct FaRowsCfg {
  static constexpr int BN = 128;
  static constexpr int CHUNK_BYTES = 128 * 128;
  static constexpr int NCHUNK = D / 64;
  static constexpr int TILE_BYTES = 128 * D * 2;
  static constexpr int NST = D == 128 ? 4 : 8;
  static constexpr int KV_OFF = 2 * TILE_BYTES;
  static constexpr int EPI_OFF = KV_OFF + NST * TILE_BYTES;  // 4 KB per softmax warp
  static constexpr int CTL_OFF = EPI_OFF + 8 * 4096;
  // q_full[2], q_empty[2], kv_full[NST], kv_empty[NST], s_full[2], p_half[4],
  // o_full[2], o_empty[2], u_full[], u_empty[], u_ask, x_full, x_empty, clc,
  // drain
  static constexpr int NBAR = 4 + 2 * NST + 2 + 4 + 2 + 2 + 2 * kUnitSlots + 5;
  static constexpr int UNIT_OFF = CTL_OFF + (NBAR * 8 + 15) / 16 * 16;
  static constexpr int CLC_OFF = UNIT_OFF + kUnitSlots * 48;
  static constexpr int END_OFF = CLC_OFF + 32;  // units handed out (or -1), then kMaxShares bits
  // Tile 1's (max, sum) of 128 rows for tile 0.
  static constexpr int X_OFF = END_OFF + (4 + kMaxShares / 8 + 15) / 16 * 16;
  static constexpr int SMEM_BYTES = X_OFF + 1024 + 1024;
  static constexpr int THREADS = 384;
  static constexpr int REG_SOFTMAX = 200, REG_OTHER = 104, REG_LAUNCH = 168;
  static constexpr int REG_NEED = 2 * 128 * REG_SOFTMAX + 128 * REG_OTHER;
  static_assert(REG_NEED <= THREADS * REG_LAUNCH, "register split exceeds the launch allocation");
  static_assert(SMEM_BYTES <= 232448, "shared memory per CTA");
  static_assert(sizeof(FaUnit) <= 48, "unit slot");
  static constexpr uint32_t O_COL = 256;
};

// Paged: a request's length in the line, per key/value head.
__device__ __forceinline__ long long request_line(const RowsParams &p, int tu, int r, int &row0, int &nq,
                                                  int &nk) {
  if (!request_rows(p, r, row0, nq, nk) || nq == 0) return 0;
  return tile_begin(max(0, nk - nq), tu, (nq + tu - 1) / tu);
}

// Paged, all 384 threads: the cuts before and behind this CTA's range.
__device__ __forceinline__ void find_range(const FaRowsParams &p, uint8_t *smem, FaCut &lo, FaCut &hi,
                                           long long &line, int &ranges) {
  constexpr int THREADS = 384, WARPS = THREADS / 32;
  const RowsParams &rp = p.rows;
  long long *sums = reinterpret_cast<long long *>(smem);  // [WARPS]
  FaCut *cuts = reinterpret_cast<FaCut *>(smem + 128);     // [2]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tu = p.tu;
  int row0 = 0, nq = 0, nk = 0;
  long long mine = 0, incl = 0, total = 0;
  auto block_scan = [&](int i0) {
    const int r = i0 + tid;
    mine = r < rp.n ? request_line(rp, tu, r, row0, nq, nk) : 0;
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    long long sum = 0;
    for (int w = 0; w < WARPS; w++) {
      if (w == warp) incl += sum;
      sum += sums[w];
    }
    return sum;
  };
  for (int i0 = 0; i0 < rp.n; i0 += THREADS) total += block_scan(i0);
  line = total * rp.Hk;
  const long long most = max(1ll, line / kRangeKeys);
  ranges = most < (long long)gridDim.x ? (int)most : (int)gridDim.x;
  const int c = blockIdx.x;
  if (tid < 2) cuts[tid] = FaCut{rp.n, 0, 0, 0, 0};
  __syncthreads();
  if (c < ranges && line > 0) {
    const long long at[2] = {cut_at(line, ranges, c), cut_at(line, ranges, c + 1)};
    long long before = 0;
    for (int i0 = 0; i0 < rp.n; i0 += THREADS) {
      long long sum = total;
      if (rp.n > THREADS) sum = block_scan(i0);
      const long long b = (before + incl - mine) * rp.Hk;
      for (int e = 0; e < 2; e++)
        if (mine > 0 && b <= at[e] && at[e] < b + mine * rp.Hk) {
          const long long y = at[e] - b, ctx = max(0, nk - nq);
          const int kvh = (int)(y / mine);
          const long long z = y - kvh * mine;
          int t0 = 0, t1 = (nq + tu - 1) / tu;  // the last tile that begins at or before z
          while (t1 - t0 > 1) {
            const int mid = (t0 + t1) >> 1;
            if (tile_begin(ctx, tu, mid) <= z) t0 = mid;
            else t1 = mid;
          }
          FaUnit un;
          unit_rows(un, tu, kvh, row0, nq, nk, t0);
          const long long into = z - tile_begin(ctx, tu, t0);
          cuts[e] = FaCut{i0 + tid, kvh, t0, cut_block(into, (un.keys + 127) / 128), at[e] - into};
        }
      before += sum;
    }
  }
  __syncthreads();
  lo = cuts[0];
  hi = cuts[1];
  __syncthreads();  // smem is free again
}

// Paged, the scheduler warp: hands the units between the cuts to
// give(i, unit), the end among them, and enters the unit that the next CTA goes
// on with.
template <typename Give>
__device__ __forceinline__ void walk_range(const FaRowsParams &p, const FaCut &lo, const FaCut &hi,
                                           long long line, int ranges, Give give) {
  const RowsParams &rp = p.rows;
  const int tu = p.tu, c = blockIdx.x;
  FaJoin join{-1, 0, 0, 0};
  FaUnit un;
  int i = 0, row0 = 0, nq = 0, nk = 0;
  bool ok = true;
  FaCut at = lo;
  if (at.r < rp.n) request_rows(rp, at.r, row0, nq, nk);
  while (ok && at.r < rp.n) {
    const bool last = at.r == hi.r && at.kvh == hi.kvh && at.tile == hi.tile;
    unit_rows(un, tu, at.kvh, row0, nq, nk, at.tile);
    un.kv_row = at.r;
    const int blocks = (un.keys + 127) / 128;
    const int end = last ? hi.blk : blocks;
    // Rows without a key are written by every CTA that comes by.
    if (at.blk < end || blocks == 0) {
      unit_blocks(un, p.tpt, at.blk, end);
      if (at.blk > 0 || end < blocks) un.part = 2 * c + (at.blk > 0 ? 0 : 1);
      if (at.blk == 0 && end < blocks) join = FaJoin{c, un.q_row, un.tokens, un.kvh};
      ok = give(i++, un);
    }
    if (last) break;
    at.blk = 0;
    if (++at.tile * tu < nq) continue;
    at.tile = 0;
    if (++at.kvh < rp.Hk) continue;
    at.kvh = 0;
    do {
      at.r++;
    } while (at.r < rp.n && request_line(rp, tu, at.r, row0, nq, nk) == 0);
  }
  un.kvh = -1;
  if (ok) give(i, un);
  if (join.last >= 0) {
    // The unit (hi's, of the request last looked at) ends in the first later
    // range whose end is at or behind the unit's. 32 ranges at a time.
    const long long ctx = max(0, nk - nq);
    const long long length = tile_begin(ctx, tu, hi.tile + 1) - tile_begin(ctx, tu, hi.tile);
    unit_rows(un, tu, hi.kvh, row0, nq, nk, hi.tile);
    const int blocks = (un.keys + 127) / 128, lane = threadIdx.x & 31;
    for (int x = c + 1; join.last == c; x += 32) {
      const int end = x + lane + 1;  // the range x + lane ends at this cut
      const long long e = end >= ranges ? length : cut_at(line, ranges, end) - hi.begin;
      const unsigned m = __ballot_sync(0xffffffffu, e >= length || cut_block(e, blocks) == blocks);
      if (m) join.last = x + __ffs(m) - 1;
    }
  }
  if ((threadIdx.x & 31) == 0) p.joins[c] = join;
}

template <int D, typename T, typename OutT, bool PAGED>
__global__ void __launch_bounds__(384, 1)
    fa_rows_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ FaRowsParams p) {
  using C = FaRowsCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t *sQ = smem, *sKV = smem + C::KV_OFF;
  uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + C::CTL_OFF);
  uint64_t *q_empty = q_full + 2;  // Q tiles take the two places in turn
  uint64_t *kv_full = q_full + 4;
  uint64_t *kv_empty = kv_full + C::NST;
  uint64_t *s_full = kv_empty + C::NST;
  uint64_t *p_half = s_full + 2;   // [t * 2 + half]
  uint64_t *o_full = p_half + 4;   // [t]
  uint64_t *o_empty = o_full + 2;  // [t]
  uint64_t *u_full = o_empty + 2;
  uint64_t *u_empty = u_full + kUnitSlots;
  uint64_t *u_ask = u_empty + kUnitSlots;
  uint64_t *x_full = u_ask + 1;
  uint64_t *x_empty = x_full + 1;
  uint64_t *clc_bar = x_empty + 1;
  uint64_t *drain = clc_bar + 1;
  auto unit_slot = [&](int i) {
    return reinterpret_cast<FaUnit *>(smem + C::UNIT_OFF + (i % kUnitSlots) * 48);
  };
  int *end_state = reinterpret_cast<int *>(smem + C::END_OFF);
  float2 *exchange = reinterpret_cast<float2 *>(smem + C::X_OFF);
  void *clc_resp = smem + C::CLC_OFF;
  uint32_t *tmem_base_slot = reinterpret_cast<uint32_t *>(smem + C::CLC_OFF + 16);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < C::NST; i++) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; t++) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[2 * t], 4);  // one arrival per softmax warp
      mbar_init(&p_half[2 * t + 1], 4);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 4);
    }
    for (int i = 0; i < kUnitSlots; i++) {
      mbar_init(&u_full[i], 1);
      mbar_init(&u_empty[i], 10);  // producer, MMA issuer, 8 softmax warps
    }
    mbar_init(u_ask, 1);
    mbar_init(x_full, 4);
    mbar_init(x_empty, 4);
    mbar_init(clc_bar, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_base_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base_slot;
  FaCut lo, hi;
  long long line = 0;
  int ranges = 1;
  if constexpr (PAGED) {
    pdl_launch_dependents();  // the join starts up as SMs get free
    griddep_wait();
  }
  if constexpr (PAGED) find_range(p, smem + C::EPI_OFF, lo, hi, line, ranges);

  // A whole warp's wait; all lanes get the same answer, also when it is given up.
  auto wait = [&](uint64_t *bar, int phase) {
    return (bool)__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag));
  };
  // The next unit of this CTA, for one warp (lane 0's arrival frees the slot).
  auto next_unit = [&](int i, FaUnit &un) {
    if (!wait(&u_full[i % kUnitSlots], i / kUnitSlots)) return false;
    un = *unit_slot(i);
    __syncwarp();
    if (lane == 0) mbar_arrive(&u_empty[i % kUnitSlots]);
    return un.kvh >= 0;
  };

  if (warp >= 8) {
    reg_dealloc<C::REG_OTHER>();
    if (warp == 8) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
      }
      const int box_rows = PAGED ? min(p.rows.page, 128) : 128;
      const int log_box = 31 - __clz(box_rows);
      const int log_page = PAGED ? 31 - __clz(p.rows.page) : 0;
      bool ok = true;
      int issued = 0, kq = 0;
      FaUnit un;
      for (int i = 0; next_unit(i, un); i++) {
        const int nblk = max(un.nb[0], un.nb[1]);
        if (nblk == 0) {
          if (lane == 0) mbar_arrive(u_ask);
          continue;
        }
        auto load_q = [&]() {
          const int tiles = un.tokens > p.tpt ? 2 : 1;
          for (int t = 0; t < tiles; t++, kq++) {
            const int slot = kq & 1;
            if (kq > 1 && !wait(&q_empty[slot], (kq >> 1) - 1)) return false;
            if (lane == 0) {
              mbar_arrive_expect_tx(&q_full[slot], C::NCHUNK * p.group * p.tpt * 128);
              for (int c = 0; c < C::NCHUNK; c++)
                tma_load_4d(sQ + slot * C::TILE_BYTES + c * C::CHUNK_BYTES, &tmQ, &q_full[slot], c * 64, 0,
                            un.q_row + t * p.tpt, un.kvh);
            }
          }
          return true;
        };
        // The first unit's Q goes ahead of its K and V; a later one's place may
        // still be in use, so its first K does not wait for that.
        const bool q_first = kq == 0;
        if (q_first && !(ok = load_q())) break;
        // Lane l loads box l: rows (l / NCHUNK) * box_rows on, columns (l % NCHUNK) * 64 on.
        const int pc = lane / C::NCHUNK, cc = lane - pc * C::NCHUNK;
        const int *trow = PAGED ? p.rows.table + (long long)un.kv_row * p.rows.table_stride : nullptr;
        auto page_at = [&](int b, bool on) {  // page of this lane's box in key block b, or 0
          const int key = b * C::BN + (pc << log_box);
          return PAGED && on && (pc << log_box) < C::BN && key < un.keys ? trow[key >> log_page] : 0;
        };
        // Step j loads K then V of block blk + j, and, if the tiles have blocks
        // of their own, of tile 1's block with either.
        const int ways = un.dual ? 2 : 1, blk1 = un.blk + un.nb[0];
        int page[2] = {page_at(un.blk, true), page_at(blk1, un.dual && un.nb[1] > 0)};
        for (int j = 0; j < nblk && ok; j++) {
          const int next[2] = {page_at(un.blk + j + 1, j + 1 < nblk),
                               page_at(blk1 + j + 1, un.dual && j + 1 < un.nb[1])};
          for (int load = 0; load < 2 * ways; load++) {
            const int kind = load / ways, way = load - kind * ways;
            if (way == 1 && j >= un.nb[1]) continue;
            if (j == 0 && load == ways && !q_first && !(ok = load_q())) break;  // behind the K
            const int key0 = ((way ? blk1 : un.blk) + j) * C::BN;
            const int valid = min(C::BN, un.keys - key0);
            const int boxes = PAGED ? ((valid + box_rows - 1) >> log_box) * C::NCHUNK : C::NCHUNK;
            int pg = way ? page[1] : page[0];
            if (PAGED && lane < boxes && (unsigned)pg >= (unsigned)p.rows.num_pages) {
              atomicOr(p.rows.err, kErrInput);  // the map reads zeros there
              pg = p.rows.num_pages;
            }
            const int slot = issued % C::NST, round = issued / C::NST;
            if (round > 0 && !(ok = wait(&kv_empty[slot], round - 1))) break;
            if (lane == 0) mbar_arrive_expect_tx(&kv_full[slot], boxes * box_rows * 128);
            __syncwarp();
            if (lane < boxes) {
              const CUtensorMap *m = kind ? &tmV : &tmK;
              uint8_t *dst = sKV + slot * C::TILE_BYTES + cc * C::CHUNK_BYTES + (pc << log_box) * 128;
              if (PAGED)
                tma_load_4d(dst, m, &kv_full[slot], cc * 64,
                            (key0 + (pc << log_box)) & (p.rows.page - 1), un.kvh, pg);
              else
                tma_load_4d(dst, m, &kv_full[slot], cc * 64, un.kv_row + key0, un.kvh, 0);
            }
            issued++;
          }
          page[0] = next[0];
          page[1] = next[1];
        }
        if (!ok) break;
        if (lane == 0) mbar_arrive(u_ask);  // the unit's loads are under way
      }
      if (*abort_flag && lane == 0) {
        // Abort path: let every armed copy land before the CTA exits.
        for (int u = kq - 2 < 0 ? 0 : kq - 2; u < kq; u++)
          mbar_wait_raw(&q_full[u & 1], (u >> 1) & 1, 100000000ull);
        for (int u = issued - C::NST < 0 ? 0 : issued - C::NST; u < issued; u++)
          mbar_wait_raw(&kv_full[u % C::NST], (u / C::NST) & 1, 100000000ull);
      }
    } else if (warp == 9) {
      // -------------------------------------------------------- MMA issuer
      constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t IDESC_S = idesc_mma_f32(128, C::BN, FMT, 0);
      constexpr uint32_t IDESC_O = idesc_mma_f32(128, D, FMT, 1);
      // One lane issues everything. A step inside a tile, or to another tile,
      // adds to the descriptor's address field (16-byte units), so a group of
      // MMAs costs its issuer little more than the instructions themselves.
      const bool leader = elect_one();
      const uint64_t q_desc = sdesc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = sdesc_sw128(smem_u32(sKV), 16, 1024);
      const uint64_t v_desc = sdesc_sw128(smem_u32(sKV), C::CHUNK_BYTES, 1024);
      constexpr uint32_t TILE = C::TILE_BYTES >> 4;
      auto commit = [&](uint64_t *bar) {
        if (leader) mma_commit(bar);
      };
      // S of Q place qt and the K in `slot`, into buffer b.
      auto issue_s = [&](int b, int qt, int slot) {
        if (leader) {
          const uint64_t qd = q_desc + qt * TILE, kd = k_desc + slot * TILE;
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++) {
            const uint32_t off = ((kk >> 2) * C::CHUNK_BYTES + (kk & 3) * 32) >> 4;
            mma_ss(tmem + b * 128, qd + off, kd + off, IDESC_S, kk > 0);
          }
          mma_commit(&s_full[b]);
        }
      };
      bool ok = true;
      int ring = 0;           // K/V tiles of this CTA's earlier units
      int kq = 0;             // Q tiles so far
      int cp[2] = {0, 0};     // key blocks of tile t so far
      int cu[2] = {0, 0};     // units of tile t so far
      FaUnit un;
      for (int i = 0; ok && next_unit(i, un); i++) {
        const int nblk = max(un.nb[0], un.nb[1]);
        if (nblk == 0) continue;
        // The Q tiles' places, taken in turn.
        const int tiles = un.dual ? 1 : 2, qs[2] = {kq & 1, (kq + 1) & 1};
        for (int t = 0; t < tiles && ok; t++) ok = wait(&q_full[(kq + t) & 1], (kq + t) >> 1);
        if (!ok) break;
        kq += tiles;
        // Rows of V behind the last key, up to the next multiple of 16, take
        // part with P = 0 and may hold anything: they are zeroed.
        auto zero_tail = [&](int slot, int left) {
          if (left >= C::BN || !(left & 15)) return;
          const int n = (16 - (left & 15)) * 8 * C::NCHUNK;
          for (int x = lane; x < n; x += 32) {
            const int c = x / (n / C::NCHUNK), y = x - c * (n / C::NCHUNK);
            *reinterpret_cast<uint4 *>(sKV + slot * C::TILE_BYTES + c * C::CHUNK_BYTES + left * 128 +
                                       y * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        };
        // O_t (+)= P_t V of step j, its first `steps` groups of 16 keys.
        auto issue_o = [&](int t, int slot, int j, int steps) {
          const uint64_t vd = v_desc + slot * TILE;
          const uint32_t o = tmem + C::O_COL + t * D, pt = tmem + t * 128;
          for (int half = 0; half < 2; half++) {
            if (!wait(&p_half[2 * t + half], cp[t])) return false;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < C::BN / 32; kk++) {
                const int ks = half * (C::BN / 32) + kk;
                if (ks < steps)
                  mma_ts(o, pt + ks * 8, vd + (ks * 2048 >> 4), IDESC_O, (j > 0 || ks > 0) ? 1u : 0u);
              }
            }
            __syncwarp();
          }
          cp[t]++;
          return true;
        };
        auto last_o = [&](int t) {
          commit(&o_full[t]);
          cu[t]++;
        };
        if (!un.dual) {
          // Step j reads K_j, V_j for both tiles; tile 0 may end before tile 1.
          if (!(ok = wait(&kv_full[ring % C::NST], ring / C::NST))) break;
          tc_fence_after();
          for (int t = 0; t < 2; t++) {
            if (un.nb[t] > 0) issue_s(t, qs[t], ring % C::NST);
            if (un.nb[t] <= 1) commit(&q_empty[qs[t]]);  // its last S
          }
          commit(&kv_empty[ring % C::NST]);
          for (int j = 0; j < nblk && ok; j++) {
            const int uV = ring + 2 * j + 1, sV = uV % C::NST;
            const int uK = uV + 1, sK = uK % C::NST;
            if (!(ok = wait(&kv_full[sV], uV / C::NST))) break;
            const int key0 = (un.blk + j) * C::BN, left = un.keys - key0;
            zero_tail(sV, left);
            bool k_ready = false;
            for (int t = 0; t < 2 && ok; t++) {
              if (j < un.nb[t]) {
                // O_t is overwritten by the unit's first product: the previous
                // epilogue must have read it.
                if (j == 0 && cu[t] > 0 && !(ok = wait(&o_empty[t], cu[t] - 1))) break;
                // 16-key steps that some row of this tile sees.
                const int seen = un.pos + min(un.tokens, (t + 1) * p.tpt) - key0;
                if (!(ok = issue_o(t, sV, j, min((min(seen, left) + 15) >> 4, C::BN / 16)))) break;
                if (j + 1 == un.nb[t]) last_o(t);
              }
              if (j + 1 < un.nb[t]) {
                if (!k_ready) {
                  if (!(ok = wait(&kv_full[sK], uK / C::NST))) break;
                  tc_fence_after();
                  k_ready = true;
                }
                issue_s(t, qs[t], sK);
                if (j + 2 == un.nb[t]) commit(&q_empty[qs[t]]);
              }
            }
            if (!ok) break;
            commit(&kv_empty[sV]);
            if (j + 1 < nblk) commit(&kv_empty[sK]);
          }
          ring += 2 * nblk;
        } else {
          // Step j reads K0 K1 V0 V1, or K0 V0 in the last of an odd number.
          auto score = [&](int t, int j) {
            const int u = ring + 4 * j + t, slot = u % C::NST;
            if (!wait(&kv_full[slot], u / C::NST)) return false;
            tc_fence_after();
            issue_s(t, qs[0], slot);
            commit(&kv_empty[slot]);
            return true;
          };
          for (int t = 0; t < 2 && ok; t++)
            if (un.nb[t] > 0) ok = score(t, 0);
          if (ok && nblk == 1) commit(&q_empty[qs[0]]);
          for (int j = 0; j < nblk && ok; j++) {
            for (int t = 0; t < 2 && ok; t++) {
              if (j < un.nb[t]) {
                const int u = ring + 4 * j + (j < un.nb[1] ? 2 + t : 1), sV = u % C::NST;
                if (!(ok = wait(&kv_full[sV], u / C::NST))) break;
                const int left = un.keys - (un.blk + j + (t ? un.nb[0] : 0)) * C::BN;
                zero_tail(sV, left);
                if (j == 0 && cu[t] > 0 && !(ok = wait(&o_empty[t], cu[t] - 1))) break;
                if (!(ok = issue_o(t, sV, j, min((left + 15) >> 4, C::BN / 16)))) break;
                commit(&kv_empty[sV]);
                if (j + 1 == un.nb[t]) last_o(t);
              }
              if (j + 1 < un.nb[t]) ok = score(t, j + 1);
            }
            if (ok && j + 2 == nblk) commit(&q_empty[qs[0]]);
          }
          ring += 2 * (un.nb[0] + un.nb[1]);
        }
      }
      // Every MMA this warp issued has completed before TMEM is released.
      commit(drain);
      mbar_wait_raw(drain, 0, 100000000ull);
    } else if (warp == 10) {
      // --------------------------------------------------------- scheduler
      FaUnit un;
      auto hand_out = [&](int i) {  // un as the CTA's i-th
        if (lane == 0) {
          *unit_slot(i) = un;
          mbar_arrive(&u_full[i % kUnitSlots]);
        }
      };
      if constexpr (PAGED) {
        walk_range(p, lo, hi, line, ranges, [&](int i, const FaUnit &next) {
          if (i >= kUnitSlots && !wait(&u_empty[i % kUnitSlots], i / kUnitSlots - 1)) return false;
          un = next;
          hand_out(i);
          return true;
        });
      } else {
        int u = blockIdx.x, asked = 0;
        // The CTAs that this one runs for, itself the first, as far as units are
        // dealt out to them: bit u % 32 of lane u / 32.
        uint32_t mine = u < p.shares && lane == u >> 5 ? 1u << (u & 31) : 0u;
        bool ok = true, have = true;
        int i = 0;
        for (;; i++) {
          if (i > 0 && !(ok = wait(u_ask, i - 1))) break;
          if (i >= kUnitSlots && !(ok = wait(&u_empty[i % kUnitSlots], i / kUnitSlots - 1))) break;
          for (bool first = i == 0;; first = false) {
            if (!first && p.dynamic) {
              if (lane == 0) {
                mbar_arrive_expect_tx(clc_bar, 16);
                clc_try_cancel(clc_resp, clc_bar);
              }
              __syncwarp();
              if (!(ok = wait(clc_bar, asked))) {
                mbar_wait_raw(clc_bar, asked & 1, 100000000ull);
                break;
              }
              asked++;
              u = clc_answer(clc_resp);
              if ((unsigned)u < (unsigned)p.shares && lane == u >> 5) mine |= 1u << (u & 31);
              fence_proxy_async_smem();
              __syncwarp();
            } else if (!first) {
              u = u < p.units - (int)gridDim.x ? u + (int)gridDim.x : -1;
            }
            have = u >= 0;
            if (!have || prompt_unit(p, u, un)) break;
          }
          if (!ok || !have) break;
          hand_out(i);
        }
        if (lane == 0) end_state[0] = ok ? i : -1;
        if (lane < kMaxShares / 32) end_state[1 + lane] = (int)mine;
        __syncwarp();
        asm volatile("bar.arrive 1, 64;" ::: "memory");
      }
    } else if (!PAGED) {  // (paged: find_range has looked at all of them)
      const bool bad = check_requests(p.rows, lane);
      // The scheduler's end, which comes whatever its own (bounded) waits end with.
      __syncwarp();
      asm volatile("bar.sync 1, 64;" ::: "memory");
      int i = end_state[0];
      bool ok = i >= 0;
      for (int share = 0; ok && bad && share < p.shares; share++)
        if (end_state[1 + (share >> 5)] >> (share & 31) & 1)
          ok = deal_units(p, share, [&](const FaUnit &un) {
            if (i >= kUnitSlots && !wait(&u_empty[i % kUnitSlots], i / kUnitSlots - 1)) return false;
            if (lane == 0) {
              *unit_slot(i) = un;
              mbar_arrive(&u_full[i % kUnitSlots]);
            }
            i++;
            return true;
          });
      if (ok && (i < kUnitSlots || wait(&u_empty[i % kUnitSlots], i / kUnitSlots - 1)) && lane == 0) {
        unit_slot(i)->kvh = -1;
        mbar_arrive(&u_full[i % kUnitSlots]);
      }
    }
  } else {
    reg_alloc<C::REG_SOFTMAX>();
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2;           // tile 0 or 1
    const int row = threadIdx.x & 127;  // row within the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + t * 128;
    const uint32_t tO = tmem + lane_off + C::O_COL + t * D;
    const float sl2 = p.scale_log2;
    bool ok = true;
    int cs = 0, cu = 0, cx = 0;  // key blocks and units of this tile, dual units so far
    for (int i = 0; ok; i++) {
      // The unit's slot is kept until its epilogue is done, which reads it
      // again: a row of scores leaves few registers.
      if (!wait(&u_full[i % kUnitSlots], i / kUnitSlots)) break;
      const FaUnit &un = *unit_slot(i);
      if (un.kvh < 0) break;
      const int nblk = un.nb[t];
      // Keys of the unit's next block that this row sees; rows that hold no
      // query are not masked.
      int valid = 0x3fffffff;
      {
        const int tok = row * p.recip >> 16, t0 = un.dual ? 0 : t * p.tpt;  // the tile's first token
        const int b0 = un.blk + (un.dual && t ? un.nb[0] : 0);
        if (tok < min(un.tokens - t0, p.tpt)) valid = un.pos + t0 + tok + 1 - b0 * C::BN;
      }
      float m_used = -INFINITY;  // log2-domain max the P values are relative to
      float l = 0.0f;
      for (int j = 0; j < nblk; j++) {
        ok = wait(&s_full[t], cs);
        if (!ok) break;
        cs++;
        tc_fence_after();
        uint32_t sbuf[128];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld32(tS + c * 32, sbuf + c * 32);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; c++) reg_fence32(sbuf + c * 32);
        const bool masked = __any_sync(0xffffffffu, valid < C::BN);
        if (masked) {
#pragma unroll
          for (int x = 0; x < 128; x++)
            if (x >= valid) sbuf[x] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 128; x += 2)
          mx[(x >> 1) & 3] = max3f(mx[(x >> 1) & 3], __uint_as_float(sbuf[x]), __uint_as_float(sbuf[x + 1]));
        // The max moves only when this block's P would pass 2^kMaxExp.
        const float m_new = max3f(mx[0], mx[1], fmaxf(mx[2], mx[3])) * sl2;
        const bool need = m_new > m_used + kMaxExp;
        if (__any_sync(0xffffffffu, need)) {
          const float m_tgt = need ? m_new - kHeadroom : m_used;
          const float factor = need ? ex2_approx(m_used - m_tgt) : 1.0f;
          l *= factor;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
              reg_fence32(o);
#pragma unroll
              for (int x = 0; x < 32; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
              tmem_st32(tO + c * 32, o);
            }
          }
          m_used = m_tgt;
        }
        // P = 2^(s*scale*log2e - m), every one by ex2 (the non-causal kernel takes
        // a quarter on the FMA pipe; here that took 8192 tokens 3 % longer, and a
        // masked score would not reach 0 there).
        uint64_t part2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
        const uint64_t sl2x2 = f2_pack(sl2, sl2);
        const float m_sub = m_used == -INFINITY ? 0.0f : m_used;  // no key so far: all P are 0
        const uint64_t neg_mx2 = f2_pack(-m_sub, -m_sub);
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const float *v = reinterpret_cast<const float *>(sbuf + c * 32);
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 16; x++) {
            const float2 e = f2_unpack(f2_fma(f2_pack(v[2 * x], v[2 * x + 1]), sl2x2, neg_mx2));
            const float p0 = ex2_approx(e.x), p1 = ex2_approx(e.y);
            part2[x & 1] = f2_add(part2[x & 1], f2_pack(p0, p1));
            pk[x] = pack16x2<T>(p0, p1);
          }
          tmem_st16(tS + c * 16, pk);
          if (c == 1 || c == 3) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[2 * t + (c == 3 ? 1 : 0)]);
          }
        }
        const float2 s0 = f2_unpack(part2[0]), s1 = f2_unpack(part2[1]);
        l += (s0.x + s0.y) + (s1.x + s1.y);
        valid -= C::BN;
      }
      if (!ok) break;
      // ------------------------------------------------------- epilogue
      if (nblk > 0) {
        ok = wait(&o_full[t], cu);
        if (!ok) break;
        cu++;
        tc_fence_after();
      }
      // Dual: tile 1 leaves its maximum and sum, and its O in TMEM, to tile 0.
      float w0 = 1.0f, w1 = 0.0f;  // weights of the own and of tile 1's O
      const bool joint = un.dual && t == 0;
      const int nblk1 = joint ? un.nb[1] : 0;
      if (un.dual) {
        if (t == 1) {
          if (cx > 0 && !(ok = wait(x_empty, cx - 1))) break;
          exchange[row] = make_float2(m_used, l);
          // (its O is complete: o_full was waited for)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(x_full);
            mbar_arrive(&u_empty[i % kUnitSlots]);
          }
          cx++;
          continue;
        }
        if (!(ok = wait(x_full, cx))) break;
        tc_fence_after();
        const float2 other = exchange[row];
        __syncwarp();
        if (lane == 0) mbar_arrive(x_empty);
        cx++;
        const float top = fmaxf(m_used, other.x);
        if (top != -INFINITY) {
          w0 = ex2_approx(m_used - top);
          w1 = ex2_approx(other.x - top);
          l = l * w0 + other.y * w1;
          m_used = top;
        } else {
          l += other.y;  // 0, or NaN
        }
      }
      const int tok = row * p.recip >> 16, head = row - tok * p.group;
      const int t0 = un.dual ? 0 : t * p.tpt;          // the tile's first token
      // A row that sees no key (a prompt's sees its own) is 0 and -inf. Scores that
      // are all -inf are l = 0 too: 0 / 0 = NaN. (A NaN score is a NaN l.)
      const int part_at = PAGED ? un.part : -1;
      const bool none = PAGED && un.pos + t0 + tok < 0;
      const float inv = part_at >= 0 ? 1.0f : none ? 0.0f : 1.0f / l;
      const float lse = none ? -INFINITY : (m_used + log2f(l)) * 0.69314718055994531f;
      w0 *= inv;
      w1 *= inv;
      const int ntok = min(un.tokens - t0, p.tpt);  // its tokens (<= 0: none)
      const bool live = tok < ntok;
      const int kvh = un.kvh, q_row = un.q_row + t0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&u_empty[i % kUnitSlots]);
      if (ntok <= 0) continue;
      // Column chunk c of this row, normalised; rows without a key are 0
      // whatever the accumulator holds.
      auto chunk = [&](int c, float *v) {
        uint32_t o[32] = {};
        if (nblk > 0) {
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
          reg_fence32(o);
          if (c == D / 32 - 1) {
            // O_t is read out: the next unit's first product may overwrite it.
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[t]);
          }
        }
#pragma unroll
        for (int x = 0; x < 32; x++) v[x] = none ? 0.0f : __uint_as_float(o[x]) * w0;
        if (nblk1 > 0) {
          tmem_ld32(tO + D + c * 32, o);
          tmem_wait_ld();
          reg_fence32(o);
          if (c == D / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[1]);
          }
#pragma unroll
          for (int x = 0; x < 32; x++) v[x] = w1 > 0.0f ? fmaf(__uint_as_float(o[x]), w1, v[x]) : v[x];
        }
      };
      if (part_at >= 0) {
        const long long r = (long long)part_at * 256 + t * 128 + row;
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
          float v[32];
          chunk(c, v);
          if (live) store_row_chunk<float>(p.part_o + r * D + c * 32, v);
        }
        if (live) p.part_ml[r] = make_float2(m_used, l);
        continue;
      }
      // Stores of whole 128-byte row segments through the warp's staging
      // block (16-byte pieces XOR-swizzled by row).
      constexpr int CPR = 128 / (int)sizeof(OutT);  // columns per round
      uint8_t *stg = smem + C::EPI_OFF + warp * 4096;
#pragma unroll
      for (int rnd = 0; rnd < D / CPR; rnd++) {
#pragma unroll
        for (int cc = 0; cc < CPR / 32; cc++) {
          float v[32];
          chunk(rnd * (CPR / 32) + cc, v);
          constexpr int PIECES = 32 * (int)sizeof(OutT) / 16;
          alignas(16) OutT pk[32];
#pragma unroll
          for (int x = 0; x < 32; x++) pk[x] = from_f32<OutT>(v[x]);
#pragma unroll
          for (int pc = 0; pc < PIECES; pc++)
            *reinterpret_cast<uint4 *>(stg + lane * 128 + (((cc * PIECES + pc) ^ (lane & 7)) << 4)) =
                reinterpret_cast<const uint4 *>(pk)[pc];
        }
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 8; it++) {
          const int pid = it * 32 + lane, r = pid >> 3, part = pid & 7;
          const uint4 val = *reinterpret_cast<const uint4 *>(stg + r * 128 + ((part ^ (r & 7)) << 4));
          const int tr = (warp & 3) * 32 + r;  // row within the tile
          const int rt = tr * p.recip >> 16;
          if (rt < ntok)
            *reinterpret_cast<uint4 *>(static_cast<OutT *>(p.rows.o) +
                                       (long long)(q_row + rt) * p.rows.os[0] +
                                       (long long)(kvh * p.group + tr - rt * p.group) * p.rows.os[1] +
                                       rnd * CPR + part * (16 / (int)sizeof(OutT))) = val;
        }
        __syncwarp();
      }
      if (p.rows.lse && live)
        p.rows.lse[(long long)(kvh * p.group + head) * p.rows.tokens + q_row + tok] = lse;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.rows.err, kErrTimeout);
}

// Joins the parts of the units that cuts fell into (paged): o = sum_s w_s o_s
// / sum_s w_s l_s with w_s = 2^(m_s - max m), parts in the order of the keys.
// (Their log-sum-exps instead of (m, l) cost a row of large scores |lse| 2^-24 of
// each weight.) One CTA per (range, 32 of its unit's rows), a warp for 4 rows, 4 parts at a time
// so that their loads overlap; lane x first finds the weight of part x.
template <int D, typename OutT>
__global__ void __launch_bounds__(256) fa_rows_join_kernel(const __grid_constant__ FaRowsParams p) {
  pdl_launch_dependents();
  griddep_wait();
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int E = D / 32, ROWS = 4, U = 4;
  const int row0 = blockIdx.y * 32 + warp * ROWS;
  const FaJoin join = p.joins[c];
  if (join.last < 0) return;
  // A warp's four rows lie in one tile; it may be empty, or behind the tokens.
  const int tok0 = (row0 >> 7) * p.tpt + ((row0 & 127) * p.recip >> 16);
  if (tok0 >= join.tokens) return;
  const int parts = join.last - c + 1;
  auto part_row = [&](int x, int i) { return (long long)(2 * (c + x) + (x == 0 ? 1 : 0)) * 256 + row0 + i; };
  float mx[ROWS], acc[ROWS][E] = {}, sum[ROWS] = {};
#pragma unroll
  for (int i = 0; i < ROWS; i++) mx[i] = -INFINITY;
  for (int x = lane; x < parts; x += 32)
#pragma unroll
    for (int i = 0; i < ROWS; i++) mx[i] = fmaxf(mx[i], p.part_ml[part_row(x, i)].x);
#pragma unroll
  for (int i = 0; i < ROWS; i++)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
  for (int x0 = 0; x0 < parts; x0 += 32) {
    float w[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const float2 e = x0 + lane < parts ? p.part_ml[part_row(x0 + lane, i)] : make_float2(-INFINITY, 0.0f);
      w[i] = e.x == -INFINITY ? 0.0f : ex2_approx(e.x - mx[i]);  // 0: adds nothing
      sum[i] += w[i] * e.y;
    }
    const int n = min(32, parts - x0);
    for (int x = 0; x < n; x += U) {
      Pack<float, E> v[U][ROWS];
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < ROWS; i++)
          v[u][i] = *reinterpret_cast<const Pack<float, E> *>(
              p.part_o + part_row(x0 + min(x + u, n - 1), i) * D + lane * E);
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
          const float f = x + u < n ? __shfl_sync(0xffffffffu, w[i], (x + u) & 31) : 0.0f;
          if (f != 0.0f)
#pragma unroll
            for (int e = 0; e < E; e++) acc[i][e] = fmaf(f, v[u][i].v[e], acc[i][e]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; i++)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int row = row0 + i, t = row >> 7, tr = row & 127;
    const int rt = tr * p.recip >> 16, tok = t * p.tpt + rt;
    if (rt >= p.tpt || tok >= join.tokens) continue;
    const float inv = 1.0f / sum[i];  // (every row of a unit that was cut sees a key)
    const int h = join.kvh * p.group + tr - rt * p.group, q_row = join.q_row + tok;
    Pack<OutT, E> out;
#pragma unroll
    for (int e = 0; e < E; e++) out.v[e] = from_f32<OutT>(acc[i][e] * inv);
    *reinterpret_cast<Pack<OutT, E> *>(static_cast<OutT *>(p.rows.o) + (long long)q_row * p.rows.os[0] +
                                       (long long)h * p.rows.os[1] + lane * E) = out;
    if (p.rows.lse && lane == 0)
      p.rows.lse[(long long)h * p.rows.tokens + q_row] = (mx[i] + log2f(sum[i])) * 0.69314718055994531f;
  }
}

}  // namespace llmr
