// Attention of few new tokens per request over a paged cache (one token each
// when decoding): at most 16 or 32 query rows per request and key/value
// head, row = token * group + head.
//
// Bound by HBM: every key and value is read once and meets few rows, so what
// counts is that all SMs stream without a pause. The blocks of 128 keys of
// all (request, key/value head) pairs are laid end to end and cut into as
// many equal ranges as there are CTAs, wherever the cuts fall: contexts of any
// mix of lengths load every SM the same. Each CTA finds its range from the
// device-side lengths with one scan, then walks it; a producer warp keeps a
// ring of 160 KB of K and V tiles in flight by TMA (one box per page), across
// the borders of requests.
//
// 16 rows fill the M of mma.sync (m16n8k16), so the products take that and not
// tcgen05, whose M = 128 would be spent on an eighth of its rows; at 16 rows
// the tensor work is a third of the time the bytes take. Of a block's 128 keys
// each of 8 warps takes 16, with its own running maximum and sum and its own
// O, so no warp waits for another until a (request, head) range ends; then the
// eight are joined through shared memory. A range that the cuts split leaves
// parts in the workspace, and the CTA that finishes last joins them, in the
// order of the keys whoever that is.
#pragma once
#include "paged_kernels.cuh"

namespace llmr {

constexpr int kDecodeCtas = 160;  // upper bound of the grid (workspace, counters)

template <int D, int MT>
struct DecodeCfg {
  static constexpr int BN = 128, WARPS = 8;
  // Two row tiles need more than the 168 registers that a ninth warp leaves
  // every thread: there the producer's warpgroup hands some over.
  static constexpr int ALL_WARPS = MT == 1 ? 9 : 12, THREADS = 32 * ALL_WARPS;
  static constexpr int REG_CONSUMER = 216, REG_PRODUCER = 72, REG_LAUNCH = 168;
  static constexpr int REG_NEED = 256 * REG_CONSUMER + 128 * REG_PRODUCER;
  static_assert(MT == 1 || REG_NEED <= THREADS * REG_LAUNCH, "register split exceeds the launch allocation");
  static constexpr int ROWS = 16 * MT;
  static constexpr int NCHUNK = D / 64;
  static constexpr int CHUNK_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = 128 * D * 2;
  static constexpr int NST = (MT == 1 ? 5 : 4) * (128 / D);
  static constexpr int MERGE_OFF = NST * TILE_BYTES;  // [8 warps][16 rows][D] fp32
  static constexpr int Q_OFF = MERGE_OFF + WARPS * 16 * D * 4;
  static constexpr int Q_BYTES = MT == 1 ? 0 : MT * (D / 16) * 32 * 16;
  static constexpr int ML_OFF = Q_OFF + Q_BYTES;  // [8 warps][ROWS] (max, sum)
  static constexpr int CTL_OFF = ML_OFF + WARPS * ROWS * 8;
  static constexpr int SMEM_BYTES = CTL_OFF + 2 * NST * 8 + 16 + 1024;
  static_assert(SMEM_BYTES <= 232448, "shared memory per CTA");
  // Floats of one part: O [ROWS][D], max and sum [ROWS].
  static constexpr int PART = ROWS * (D + 2);
};

struct DecodeParams {
  RowsParams rows;
  int group;
  float scale_log2;
  float *parts;   // [CTA][2][PART]
  int *counters;  // [CTA], 0 between launches
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                  uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four 8x8 16-bit matrices from shared memory; lane l gives the address of row
// l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Where CTA c of g begins in a line of `total` blocks, and who has block x.
__host__ __device__ __forceinline__ long long range_begin(long long total, int g, int c) {
  return total * c / g;
}
__host__ __device__ __forceinline__ int range_owner(long long total, int g, long long x) {
  return (int)(((x + 1) * g - 1) / total);
}

// One request as the walk meets it.
struct DecodeSeg {
  int r, row0, nq, nk, blocks;  // request, its first query row, rows, keys, key blocks
  int kvh, blk;                 // key/value head and first block of the range's next piece
};

// A request's blocks per key/value head; one for rows without a key (they are
// written too), none for a request without rows.
__device__ __forceinline__ int decode_blocks(const RowsParams &p, int r, int &row0, int &nq, int &nk) {
  if (!request_rows(p, r, row0, nq, nk) || nq == 0) return 0;
  return max(1, (nk + 127) / 128);
}

// Row r of a (request, head), columns col .. col + 3: acc / l to the output,
// and the row's log-sum-exp. A row without a key is 0 and -inf.
template <int D, typename OutT>
__device__ __forceinline__ void finish_row(const DecodeParams &p, const DecodeSeg &sg, int r, int col,
                                           const float4 &acc, float top, float l) {
  const int tok = r / p.group, h = sg.kvh * p.group + r - tok * p.group;
  const long long row = sg.row0 + tok;
  const bool none = top == -INFINITY;
  const float inv = none ? 0.0f : 1.0f / l;
  Pack<OutT, 4> out;
  out.v[0] = from_f32<OutT>(none ? 0.0f : acc.x * inv);
  out.v[1] = from_f32<OutT>(none ? 0.0f : acc.y * inv);
  out.v[2] = from_f32<OutT>(none ? 0.0f : acc.z * inv);
  out.v[3] = from_f32<OutT>(none ? 0.0f : acc.w * inv);
  *reinterpret_cast<Pack<OutT, 4> *>(static_cast<OutT *>(p.rows.o) + row * p.rows.os[0] +
                                     h * p.rows.os[1] + col) = out;
  if (p.rows.lse && col == 0)
    p.rows.lse[(long long)h * p.rows.tokens + row] =
        none ? -INFINITY : (top + log2f(l)) * 0.69314718055994531f;
}

template <int D, int MT, typename T, typename OutT>
__global__ void __launch_bounds__(DecodeCfg<D, MT>::THREADS, 1)
    fa_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ DecodeParams p) {
  using C = DecodeCfg<D, MT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  float *merge = reinterpret_cast<float *>(smem + C::MERGE_OFF);
  float2 *ml = reinterpret_cast<float2 *>(smem + C::ML_OFF);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::CTL_OFF);
  uint64_t *empty = full + C::NST;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(empty + C::NST);
  volatile int *last_flag = abort_flag + 1;
  __shared__ long long scan[C::ALL_WARPS];
  __shared__ DecodeSeg start;

  const RowsParams &rp = p.rows;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < C::NST; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], C::WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  // ------------------------------------------------ the line of blocks, my range
  // Sum of the requests' blocks in [i0, i0 + THREADS), and this thread's
  // inclusive prefix within it.
  auto block_scan = [&](int i0, long long &incl, int &mine, int &row0, int &nq, int &nk) {
    const int r = i0 + tid;
    mine = r < rp.n ? decode_blocks(rp, r, row0, nq, nk) : 0;
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    __syncthreads();  // the previous round's reads of scan[]
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    long long sum = 0;
#pragma unroll
    for (int w = 0; w < C::ALL_WARPS; w++) {
      if (w == warp) incl += sum;
      sum += scan[w];
    }
    return sum;
  };
  long long incl, total = 0;
  int mine, row0, nq, nk;
  for (int i0 = 0; i0 < rp.n; i0 += C::THREADS) total += block_scan(i0, incl, mine, row0, nq, nk);
  const long long line = total * rp.Hk;
  const int ctas = line < (long long)gridDim.x ? (int)line : (int)gridDim.x;
  const int cta = blockIdx.x;
  if (cta >= ctas) return;
  const long long lo = range_begin(line, ctas, cta), hi = range_begin(line, ctas, cta + 1);
  {
    long long before = 0;
    for (int i0 = 0; i0 < rp.n; i0 += C::THREADS) {
      long long sum = total;
      if (rp.n > C::THREADS) sum = block_scan(i0, incl, mine, row0, nq, nk);
      // Requests lie end to end as [before + incl - mine, before + incl) * Hk.
      const long long b = (before + incl - mine) * rp.Hk;
      if (mine > 0 && b <= lo && lo < (before + incl) * rp.Hk) {
        start.r = i0 + tid;
        start.row0 = row0;
        start.nq = nq;
        start.nk = nk;
        start.blocks = mine;
        start.kvh = (int)((lo - b) / mine);
        start.blk = (int)((lo - b) % mine);
      }
      before += sum;
      if (before * rp.Hk > lo) break;
    }
  }
  __syncthreads();
  DecodeSeg sg = start;
  // The next (request, key/value head); false behind the last request.
  auto advance = [&]() {
    sg.blk = 0;
    if (++sg.kvh < rp.Hk) return true;
    sg.kvh = 0;
    while (++sg.r < rp.n) {
      sg.blocks = decode_blocks(rp, sg.r, sg.row0, sg.nq, sg.nk);
      if (sg.blocks > 0) return true;
    }
    return false;
  };
  auto wait = [&](uint64_t *bar, int phase) {
    return (bool)__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag));
  };

  if (warp >= C::WARPS) {
    // -------------------------------------------------------------- producer
    if constexpr (MT > 1) reg_dealloc<C::REG_PRODUCER>();
    if (warp > C::WARPS) return;
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int box_rows = min(rp.page, 128);
    const int log_box = 31 - __clz(box_rows), log_page = 31 - __clz(rp.page);
    const int pc = lane / C::NCHUNK, cc = lane - pc * C::NCHUNK;
    bool ok = true;
    int issued = 0;
    for (long long at = lo; ok && at < hi;) {
      const int cnt = (int)min((long long)(sg.blocks - sg.blk), hi - at);
      const int *trow = rp.table + (long long)sg.r * rp.table_stride;
      auto page_at = [&](int j) {  // page of this lane's box in block j, or 0
        const int key = (sg.blk + j) * C::BN + (pc << log_box);
        return j < cnt && (pc << log_box) < C::BN && key < sg.nk ? trow[key >> log_page] : 0;
      };
      int page = page_at(0);
      for (int j = 0; j < cnt && ok; j++) {
        const int next_page = page_at(j + 1);
        const int key0 = (sg.blk + j) * C::BN;
        const int valid = max(0, min(C::BN, sg.nk - key0));
        const int boxes = ((valid + box_rows - 1) >> log_box) * C::NCHUNK;
        if (lane < boxes && (unsigned)page >= (unsigned)rp.num_pages) {
          atomicOr(rp.err, kErrInput);  // the map reads zeros there
          page = rp.num_pages;
        }
        for (int kind = 0; kind < 2; kind++) {
          const int slot = issued % C::NST, round = issued / C::NST;
          if (round > 0 && !(ok = wait(&empty[slot], round - 1))) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[slot], boxes * box_rows * 128);
          __syncwarp();
          if (lane < boxes)
            tma_load_4d(smem + slot * C::TILE_BYTES + cc * C::CHUNK_BYTES + (pc << log_box) * 128,
                        kind ? &tmV : &tmK, &full[slot], cc * 64,
                        (key0 + (pc << log_box)) & (rp.page - 1), sg.kvh, page);
          issued++;
        }
        page = next_page;
      }
      at += cnt;
      if (at < hi && !advance()) break;
    }
    if (!ok && lane == 0)  // every armed copy lands before the CTA exits
      for (int u = max(0, issued - C::NST); u < issued; u++)
        mbar_wait_raw(&full[u % C::NST], (u / C::NST) & 1, 100000000ull);
  } else {
    // -------------------------------------------------------------- consumers
    // A wait that gives up leaves its warp in the loop, so that the barriers
    // below stay matched; every later wait gives up at once.
    if constexpr (MT > 1) reg_alloc<C::REG_CONSUMER>();
    const int qa = lane >> 2, qc = (lane & 3) * 2;  // fragment row and column
    const uint32_t ring = smem_u32(smem);
    // ldmatrix rows. K: matrices (keys 0-7 | 8-15) x (d 0-7 | 8-15), d fastest;
    // V (transposed): keys fastest. Row r of a tile is 128 bytes per chunk of 64
    // columns, its 16-byte pieces XORed with r % 8.
    const int krow = warp * 16 + ((lane >> 4) << 3) + (lane & 7), kpiece = (lane >> 3) & 1;
    const int vrow = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), vpiece = lane >> 4;
    int used = 0;  // K/V tiles so far
    for (long long at = lo; at < hi;) {
      const int cnt = (int)min((long long)(sg.blocks - sg.blk), hi - at);
      const int nrows = sg.nq * p.group;
      // Q as A fragments: rows qa and qa + 8, columns qc, qc + 1 and + 8.
      auto q_word = [&](int m, int kk, int i) {
        const int r = m * 16 + qa + (i & 1) * 8, col = kk * 16 + qc + (i >> 1) * 8;
        if (r >= nrows) return 0u;
        const int tok = r / p.group, g = r - tok * p.group;
        return *reinterpret_cast<const uint32_t *>(
            static_cast<const T *>(rp.q) + (long long)(sg.row0 + tok) * rp.qs[0] +
            (long long)(sg.kvh * p.group + g) * rp.qs[1] + col);
      };
      uint32_t qf[MT == 1 ? D / 16 : 1][4];
      uint4 *sq = reinterpret_cast<uint4 *>(smem + C::Q_OFF);
      if constexpr (MT == 1) {
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++)
#pragma unroll
          for (int i = 0; i < 4; i++) qf[kk][i] = q_word(0, kk, i);
      } else {
        // (the previous range's reads are behind its last barrier)
        for (int f = warp; f < MT * (D / 16); f += C::WARPS) {
          const int m = f / (D / 16), kk = f - m * (D / 16);
          sq[f * 32 + lane] = make_uint4(q_word(m, kk, 0), q_word(m, kk, 1), q_word(m, kk, 2), q_word(m, kk, 3));
        }
        named_barrier(1, 32 * C::WARPS);
      }
      float o[MT][D / 8][4];
      float mx[MT][2], sum[MT][2];
      int lim[MT][2];  // keys the fragment's two rows see
#pragma unroll
      for (int m = 0; m < MT; m++) {
#pragma unroll
        for (int n = 0; n < D / 8; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[m][n][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          mx[m][i] = -INFINITY;
          sum[m][i] = 0.0f;
          lim[m][i] = min(sg.nk, sg.nk - sg.nq + 1 + (m * 16 + qa + i * 8) / p.group);
        }
      }
      for (int j = 0; j < cnt; j++) {
        const int key0 = (sg.blk + j) * C::BN;
        const int kslot = used % C::NST;
        wait(&full[kslot], used / C::NST);
        float s[MT][2][4] = {};
        {
          const uint32_t tile = ring + kslot * C::TILE_BYTES + krow * 128;
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++) {
            uint32_t b[4];
            ldmatrix4(b, tile + (kk >> 2) * C::CHUNK_BYTES + ((((kk & 3) * 2 + kpiece) ^ (krow & 7)) << 4));
#pragma unroll
            for (int m = 0; m < MT; m++) {
              if constexpr (MT == 1) {
                mma_16816<T>(s[m][0], qf[kk], b[0], b[1]);
                mma_16816<T>(s[m][1], qf[kk], b[2], b[3]);
              } else {
                const uint4 f = sq[(m * (D / 16) + kk) * 32 + lane];
                const uint32_t a[4] = {f.x, f.y, f.z, f.w};
                mma_16816<T>(s[m][0], a, b[0], b[1]);
                mma_16816<T>(s[m][1], a, b[2], b[3]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[kslot]);
        used++;
        const int k0 = key0 + warp * 16 + qc;  // this lane's first key
        const bool tail = key0 + C::BN > sg.nk - sg.nq + 1;  // some row may not see all keys
        uint32_t pf[MT][4];
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
          for (int i = 0; i < 2; i++) {  // rows qa, qa + 8
            float x[4] = {s[m][0][2 * i], s[m][0][2 * i + 1], s[m][1][2 * i], s[m][1][2 * i + 1]};
            if (tail) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (k0 + (e >> 1) * 8 + (e & 1) >= lim[m][i]) x[e] = -INFINITY;
            }
            float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * p.scale_log2;
            // The maximum moves only when this block passes it by 2^15, the
            // most an fp16 P may hold.
            const bool need = top > mx[m][i] + 15.0f;
            if (__any_sync(0xffffffffu, need)) {
              const float f = need ? ex2_approx(mx[m][i] - top) : 1.0f;
              if (need) mx[m][i] = top;
              sum[m][i] *= f;
#pragma unroll
              for (int n = 0; n < D / 8; n++) {
                o[m][n][2 * i] *= f;
                o[m][n][2 * i + 1] *= f;
              }
            }
            const float sub = mx[m][i] == -INFINITY ? 0.0f : mx[m][i];  // no key so far: all P are 0
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = ex2_approx(fmaf(x[e], p.scale_log2, -sub));
            sum[m][i] += (x[0] + x[1]) + (x[2] + x[3]);
            pf[m][i] = pack16x2<T>(x[0], x[1]);
            pf[m][i + 2] = pack16x2<T>(x[2], x[3]);
          }
        }
        const int vslot = used % C::NST;
        wait(&full[vslot], used / C::NST);
        const uint32_t tile = ring + vslot * C::TILE_BYTES + vrow * 128;
        // Values behind the last key may be anything: they count as 0.
        const bool cut = key0 + C::BN > sg.nk;
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (cut) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int k = k0 + i * 8;
            keep[i] = k + 1 < sg.nk ? 0xffffffffu : k < sg.nk ? 0xffffu : 0u;
          }
        }
#pragma unroll
        for (int n2 = 0; n2 < D / 16; n2++) {
          uint32_t b[4];
          ldmatrix4_trans(b, tile + (n2 >> 2) * C::CHUNK_BYTES + ((((n2 & 3) * 2 + vpiece) ^ (vrow & 7)) << 4));
          if (cut) {
            b[0] &= keep[0];
            b[1] &= keep[1];
            b[2] &= keep[0];
            b[3] &= keep[1];
          }
#pragma unroll
          for (int m = 0; m < MT; m++) {
            mma_16816<T>(o[m][2 * n2], pf[m], b[0], b[1]);
            mma_16816<T>(o[m][2 * n2 + 1], pf[m], b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[vslot]);
        used++;
      }
      // ------------------------------------------ the eight warps' results joined
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float t = sum[m][i];
          t += __shfl_xor_sync(0xffffffffu, t, 1);
          t += __shfl_xor_sync(0xffffffffu, t, 2);
          if ((lane & 3) == 0) ml[warp * C::ROWS + m * 16 + qa + i * 8] = make_float2(mx[m][i], t);
        }
      named_barrier(1, 32 * C::WARPS);
      const bool whole = sg.blk == 0 && cnt == sg.blocks;
      float *part = p.parts + (long long)(2 * cta + (sg.blk > 0 ? 0 : 1)) * C::PART;
#pragma unroll
      for (int m = 0; m < MT; m++) {
        if (m * 16 >= nrows) break;
        // The rows' common maximum; each warp's O is brought to it.
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int r = m * 16 + qa + i * 8;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < C::WARPS; w++) top = fmaxf(top, ml[w * C::ROWS + r].x);
          const float f = mx[m][i] == -INFINITY ? 0.0f : ex2_approx(mx[m][i] - top);
          float *row = merge + (warp * 16 + qa + i * 8) * D;
          if (r < nrows) {
#pragma unroll
            for (int n = 0; n < D / 8; n++)
              *reinterpret_cast<float2 *>(row + ((n * 8 + qc) ^ (qa << 3))) =
                  make_float2(o[m][n][2 * i] * f, o[m][n][2 * i + 1] * f);
          }
        }
        named_barrier(1, 32 * C::WARPS);
        for (int x = tid; x < 16 * (D / 4); x += 32 * C::WARPS) {
          const int rr = x / (D / 4), col = (x - rr * (D / 4)) * 4, r = m * 16 + rr;
          if (r >= nrows) break;
          float top = -INFINITY, l = 0.0f;
#pragma unroll
          for (int w = 0; w < C::WARPS; w++) top = fmaxf(top, ml[w * C::ROWS + r].x);
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < C::WARPS; w++) {
            const float2 e = ml[w * C::ROWS + r];
            if (e.x != -INFINITY) l += e.y * ex2_approx(e.x - top);
            const float4 v = *reinterpret_cast<const float4 *>(merge + (w * 16 + rr) * D + (col ^ ((rr & 7) << 3)));
            acc.x += v.x;
            acc.y += v.y;
            acc.z += v.z;
            acc.w += v.w;
          }
          if (whole)
            finish_row<D, OutT>(p, sg, r, col, acc, top, l);
          else {
            __stcg(reinterpret_cast<float4 *>(part + r * D + col), acc);
            if (col == 0) __stcg(reinterpret_cast<float2 *>(part + C::ROWS * D) + r, make_float2(top, l));
          }
        }
        named_barrier(1, 32 * C::WARPS);  // merge (and, at the end, ml) may be written again
      }
      if (!whole) {
        // Parts of this (request, head): CTAs first .. last of the line.
        const long long b0 = at - sg.blk;
        const int first = range_owner(line, ctas, b0);
        const int last = range_owner(line, ctas, b0 + sg.blocks - 1);
        __threadfence();
        named_barrier(1, 32 * C::WARPS);
        if (tid == 0) *last_flag = atomicAdd(p.counters + first, 1) == last - first;
        named_barrier(1, 32 * C::WARPS);
        if (*last_flag) {
          __threadfence();
          for (int x = tid; x < nrows * (D / 4); x += 32 * C::WARPS) {
            const int r = x / (D / 4), col = (x - r * (D / 4)) * 4;
            auto at_part = [&](int c) { return p.parts + (long long)(2 * c + (c == first ? 1 : 0)) * C::PART; };
            float top = -INFINITY, l = 0.0f;
#pragma unroll 4
            for (int c = first; c <= last; c++)
              top = fmaxf(top, __ldcg(reinterpret_cast<const float2 *>(at_part(c) + C::ROWS * D) + r).x);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int c = first; c <= last; c++) {
              const float2 e = __ldcg(reinterpret_cast<const float2 *>(at_part(c) + C::ROWS * D) + r);
              const float4 v = __ldcg(reinterpret_cast<const float4 *>(at_part(c) + r * D + col));
              const float f = e.x == -INFINITY ? 0.0f : ex2_approx(e.x - top);
              l = fmaf(e.y, f, l);
              acc.x = fmaf(v.x, f, acc.x);
              acc.y = fmaf(v.y, f, acc.y);
              acc.z = fmaf(v.z, f, acc.z);
              acc.w = fmaf(v.w, f, acc.w);
            }
            finish_row<D, OutT>(p, sg, r, col, acc, top, l);
          }
          if (tid == 0) p.counters[first] = 0;
        }
        named_barrier(1, 32 * C::WARPS);  // last_flag may be written again
      }
      at += cnt;
      if (at < hi && !advance()) break;
    }
    if (tid == 0 && *abort_flag) atomicOr(rp.err, kErrTimeout);
  }
}

}  // namespace llmr
