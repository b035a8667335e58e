// Attention of few new tokens per request over a paged cache (one token each
// when decoding): at most 32 query rows per request and key/value head,
// row = token * group + head.
//
// Bound by HBM: 64 decodes over 127k keys, 32 / 8 heads of 128, take 87 us of
// device time = 6.0 TB/s (91 % of a plain copy's rate; 89 us per call, back to
// back), 32 requests of 32 rows over 4096 keys 95 us. Every key and value is read once and meets few rows, so what
// counts is that all SMs stream without a pause. The blocks of 64 keys of all
// (request, key/value head) pairs are laid end to end and cut into as many
// equal ranges as there are CTAs, wherever the cuts fall: contexts of any mix of
// lengths load every SM the same. A pair counts kPairBlocks more than its
// blocks, for its queries' way in and its result's way out. Each CTA finds its range
// from the device-side lengths with one scan, then walks it; a producer warp
// keeps a ring of K and V tiles in flight by TMA (one box per page), across
// the borders of requests. Two CTAs share an SM, so one streams while the other
// ends a pair (with one CTA of twice the size, SMs whose range held many short
// contexts took a third longer than the rest).
//
// 16 rows fill the M of mma.sync (m16n8k16), so the products take that and not
// tcgen05, whose M = 128 would be spent on a few of its rows. The four warps
// are RW row tiles of 16 times KW shares of a block's keys: (1, 4) up to 16
// rows, (2, 2) up to 32. Every warp has its own running
// maximum and sum and its own O, so none waits for another until a pair's
// range ends; then the KW shares are joined through shared memory. A pair
// that the cuts split leaves parts in the workspace, which a second launch
// joins in the order of the keys.
#pragma once
#include <type_traits>

#include "paged_rows.cuh"

namespace llmr {

constexpr int kDecodeCtas = 320;  // upper bound of the grid (workspace)
constexpr int kPairBlocks = 2;    // what a pair costs besides its blocks, in blocks
constexpr int kRangeBlocks = 2;  // least length of a CTA's range
constexpr int kDecodeBN = 64;     // keys per block

template <int D, int RW>
struct DecodeCfg {
  static constexpr int BN = kDecodeBN, WARPS = 4, THREADS = 32 * (WARPS + 1);
  static_assert(RW == 1 || RW == 2, "one or two row tiles");
  static constexpr int KW = WARPS / RW, KEYS = BN / KW;  // a warp's keys of a block
  static constexpr int ROWS = 16 * RW;
  static constexpr int NCHUNK = D / 64;
  static constexpr int CHUNK_BYTES = BN * 128;
  static constexpr int TILE_BYTES = BN * D * 2;
  static constexpr int MERGE_BYTES = WARPS * 16 * D * 4;  // [warp][16 rows][D] fp32
  static constexpr int NST = 4 * (128 / D);
  static constexpr int MERGE_OFF = NST * TILE_BYTES;
  static constexpr int ML_OFF = MERGE_OFF + MERGE_BYTES;  // [warp][16] (max, sum)
  static constexpr int CTL_OFF = ML_OFF + WARPS * 16 * 8;
  static constexpr int SMEM_BYTES = CTL_OFF + 2 * NST * 8 + 16 + 1024;
  static_assert(SMEM_BYTES <= 233472 / 2 - 1024 - 256, "shared memory for two CTAs per SM");
  // Floats of one part: O [ROWS][D], max and sum [ROWS].
  static constexpr int PART = ROWS * (D + 2);
};

// A pair that a cut falls into, entered by the CTA that begins it.
struct DecodeJoin {
  int last;  // CTA of its last part; -1: this CTA begins no such pair
  int row0, nq, kvh;
};

struct DecodeParams {
  RowsParams rows;
  int group;
  float scale_log2;
  float *parts;       // [CTA][2][PART]
  DecodeJoin *joins;  // [CTA]
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

// One pair as the walk meets it.
struct DecodeSeg {
  int r, row0, nq, nk, blocks;  // request, its first query row, rows, keys, key blocks
  int kvh;                      // key/value head
  int at;                       // where the pair begins, counted from the CTA's range
};

// A request's length in the line per key/value head: its blocks (one for rows
// without a key: they are written too) and kPairBlocks; 0 for a request without
// rows.
__device__ __forceinline__ int decode_blocks(bool ok, int nq, int nk) {
  return ok && nq > 0 ? max(1, (nk + kDecodeBN - 1) / kDecodeBN) + kPairBlocks : 0;
}

// Row r of a pair, columns col ..: acc / l to the output, and the row's
// log-sum-exp. A row that sees no key is 0 and -inf; one whose scores are all
// -inf has l = 0 too, and is 0 / 0 = NaN and -inf; a NaN score is a NaN l.
__device__ __forceinline__ float elem(const float2 &v, int i) { return i ? v.y : v.x; }
__device__ __forceinline__ float elem(const float4 &v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
template <int D, typename OutT, typename Acc>
__device__ __forceinline__ void finish_row(const DecodeParams &p, const DecodeSeg &sg, int r, int col,
                                           const Acc &acc, float top, float l) {
  constexpr int N = sizeof(Acc) / 4;
  const int tok = r / p.group, h = sg.kvh * p.group + r - tok * p.group;
  const long long row = sg.row0 + tok;
  const bool none = sg.nk - sg.nq + tok < 0;
  const float inv = 1.0f / l;
  Pack<OutT, N> out;
#pragma unroll
  for (int i = 0; i < N; i++) out.v[i] = from_f32<OutT>(none ? 0.0f : elem(acc, i) * inv);
  *reinterpret_cast<Pack<OutT, N> *>(static_cast<OutT *>(p.rows.o) + row * p.rows.os[0] +
                                     h * p.rows.os[1] + col) = out;
  if (p.rows.lse && col == 0)
    p.rows.lse[(long long)h * p.rows.tokens + row] =
        none ? -INFINITY : (top + log2f(l)) * 0.69314718055994531f;
}

template <int D, int RW, typename T, typename OutT>
__global__ void __launch_bounds__(DecodeCfg<D, RW>::THREADS, 2)
    fa_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ DecodeParams p) {
  using C = DecodeCfg<D, RW>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  float *merge = reinterpret_cast<float *>(smem + C::MERGE_OFF);
  float2 *ml = reinterpret_cast<float2 *>(smem + C::ML_OFF);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::CTL_OFF);
  uint64_t *empty = full + C::NST;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(empty + C::NST);
  __shared__ long long scan[C::WARPS + 1];
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
  pdl_launch_dependents();  // the join's CTAs fit beside this kernel's and wait there
  griddep_wait();
  // ------------------------------------------------ the line of blocks, my range
  // Each thread takes R neighbouring requests: the sum of all lengths from i0
  // on (STRIDE requests), and the place of this thread's first.
  constexpr int R = 4, STRIDE = R * C::THREADS;
  int size[R], row0[R], nq[R], nk[R];
  auto block_scan = [&](int i0, long long &begin) {
    int a[R], e[R], k[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int r = min(i0 + tid * R + i, rp.n - 1);
      a[i] = rp.cu[r];
      e[i] = rp.cu[r + 1];
      k[i] = rp.kv_lens[r];
    }
    long long mine = 0;
#pragma unroll
    for (int i = 0; i < R; i++) {
      size[i] = i0 + tid * R + i < rp.n
                    ? decode_blocks(check_rows(rp, a[i], e[i], k[i], row0[i], nq[i], nk[i]), nq[i], nk[i])
                    : 0;
      mine += size[i];
    }
    long long incl = mine;
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
    for (int w = 0; w <= C::WARPS; w++) {
      if (w == warp) incl += sum;
      sum += scan[w];
    }
    begin = incl - mine;
    return sum;
  };
  long long begin, total = 0;
  for (int i0 = 0; i0 < rp.n; i0 += STRIDE) total += block_scan(i0, begin);
  const long long line = total * rp.Hk;
  const long long most = max(1ll, line / kRangeBlocks);
  const int ctas = line == 0 ? 0 : most < (long long)gridDim.x ? (int)most : (int)gridDim.x;
  const int cta = blockIdx.x;
  if (tid == 0) p.joins[cta].last = -1;
  if (cta >= ctas) return;
  const long long lo = range_begin(line, ctas, cta), hi = range_begin(line, ctas, cta + 1);
  {
    long long before = 0;
    for (int i0 = 0; i0 < rp.n; i0 += STRIDE) {
      long long sum = total;
      if (rp.n > STRIDE) sum = block_scan(i0, begin);
      // Requests lie end to end, each rp.Hk times its length.
      long long b = (before + begin) * rp.Hk;
#pragma unroll
      for (int i = 0; i < R; i++) {
        const long long e = b + (long long)size[i] * rp.Hk;
        if (b <= lo && lo < e) {
          start.r = i0 + tid * R + i;
          start.row0 = row0[i];
          start.nq = nq[i];
          start.nk = nk[i];
          start.blocks = size[i] - kPairBlocks;
          start.kvh = (int)((lo - b) / size[i]);
          start.at = (int)(b + (long long)start.kvh * size[i] - lo);
        }
        b = e;
      }
      before += sum;
      if (before * rp.Hk > lo) break;
    }
  }
  __syncthreads();
  DecodeSeg sg = start;
  const int len = (int)(hi - lo);
  // My blocks [b0, b0 + cnt) of the current pair.
  auto piece = [&](int &b0, int &cnt) {
    const int first = sg.at + kPairBlocks;
    b0 = max(0, -first);
    cnt = max(0, min(sg.blocks, len - first) - b0);
  };
  // The next pair; false behind the range.
  auto advance = [&]() {
    sg.at += sg.blocks + kPairBlocks;
    if (sg.at >= len) return false;
    if (++sg.kvh < rp.Hk) return true;
    sg.kvh = 0;
    while (++sg.r < rp.n) {
      const bool ok = request_rows(rp, sg.r, sg.row0, sg.nq, sg.nk);
      sg.blocks = decode_blocks(ok, sg.nq, sg.nk) - kPairBlocks;
      if (sg.blocks > 0) return true;
    }
    return false;
  };
  auto wait = [&](uint64_t *bar, int phase) {
    return (bool)__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, abort_flag));
  };

  if (warp == C::WARPS) {
    // -------------------------------------------------------------- producer
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int box_rows = min(rp.page, C::BN);
    const int log_box = 31 - __clz(box_rows), log_page = 31 - __clz(rp.page);
    const int pc = lane / C::NCHUNK, cc = lane - pc * C::NCHUNK;
    bool ok = true;
    int issued = 0;
    do {
      int b0, cnt;
      piece(b0, cnt);
      const int *trow = rp.table + (long long)sg.r * rp.table_stride;
      auto page_at = [&](int j) {  // page of this lane's box in block j, or 0
        const int key = (b0 + j) * C::BN + (pc << log_box);
        return j < cnt && (pc << log_box) < C::BN && key < sg.nk ? trow[key >> log_page] : 0;
      };
      int page = page_at(0);
      for (int j = 0; j < cnt && ok; j++) {
        const int next_page = page_at(j + 1);
        const int key0 = (b0 + j) * C::BN;
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
    } while (ok && advance());
    if (!ok && lane == 0)  // every armed copy lands before the CTA exits
      for (int u = max(0, issued - C::NST); u < issued; u++)
        mbar_wait_raw(&full[u % C::NST], (u / C::NST) & 1, 100000000ull);
    return;
  }
  // ---------------------------------------------------------------- consumers
  // A wait that gives up leaves its warp in the loop, so that the barriers
  // below stay matched; every later wait gives up at once.
  const int rw = warp / C::KW, kw = warp - rw * C::KW;  // row tile, share of the keys
  const int qa = lane >> 2, qc = (lane & 3) * 2;        // fragment row and column
  const uint32_t ring = smem_u32(smem);
  // ldmatrix rows. K: matrices (keys 0-7 | 8-15) x (d 0-7 | 8-15), d fastest;
  // V (transposed): keys fastest. Row r of a tile is 128 bytes per chunk of 64
  // columns, its 16-byte pieces XORed with r % 8.
  const int krow = kw * C::KEYS + ((lane >> 4) << 3) + (lane & 7), kpiece = (lane >> 3) & 1;
  const int vrow = kw * C::KEYS + (((lane >> 3) & 1) << 3) + (lane & 7), vpiece = lane >> 4;
  int used = 0;  // K/V tiles so far
  do {
    int b0, cnt;
    piece(b0, cnt);
    if (cnt == 0) continue;
    const int nrows = sg.nq * p.group;
    const bool idle = rw * 16 >= nrows;  // a row tile without rows
    // Q as A fragments: rows qa and qa + 8, columns qc, qc + 1 and + 8.
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int r = rw * 16 + qa + i * 8;
      const int tok = r / p.group, g = r - tok * p.group;
      const T *src = static_cast<const T *>(rp.q) + (long long)(sg.row0 + tok) * rp.qs[0] +
                     (long long)(sg.kvh * p.group + g) * rp.qs[1] + qc;
#pragma unroll
      for (int kk = 0; kk < D / 16; kk++) {
        qf[kk][i] = r < nrows ? *reinterpret_cast<const uint32_t *>(src + kk * 16) : 0u;
        qf[kk][i + 2] = r < nrows ? *reinterpret_cast<const uint32_t *>(src + kk * 16 + 8) : 0u;
      }
    }
    float o[D / 8][4] = {};
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    int lim[2];  // keys the fragment's two rows see
#pragma unroll
    for (int i = 0; i < 2; i++)
      lim[i] = min(sg.nk, sg.nk - sg.nq + 1 + (rw * 16 + qa + i * 8) / p.group);
    for (int j = 0; j < cnt; j++) {
      const int key0 = (b0 + j) * C::BN;
      const int kslot = used % C::NST;
      wait(&full[kslot], used / C::NST);
      const int vslot = (used + 1) % C::NST;
      const bool tail = key0 + C::BN > sg.nk - sg.nq + 1;  // some row may not see all keys
      const bool cut = key0 + C::BN > sg.nk;                // some key is behind the last
      if (idle) wait(&full[vslot], (used + 1) / C::NST);
      if (!idle) {
        const int k0 = key0 + kw * C::KEYS + qc;  // this lane's first key
        float s[C::KEYS / 8][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++)
#pragma unroll
          for (int h = 0; h < C::KEYS / 16; h++) {
            uint32_t b[4];
            ldmatrix4(b, ring + kslot * C::TILE_BYTES + (krow + h * 16) * 128 + (kk >> 2) * C::CHUNK_BYTES +
                             ((((kk & 3) * 2 + kpiece) ^ (krow & 7)) << 4));
            mma_16816<T>(s[2 * h], qf[kk], b[0], b[1]);
            mma_16816<T>(s[2 * h + 1], qf[kk], b[2], b[3]);
          }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[kslot]);
        uint32_t pf[C::KEYS / 16][4];
#pragma unroll
        for (int i = 0; i < 2; i++) {  // rows qa, qa + 8
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < C::KEYS / 8; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float &x = s[n][2 * i + e];
              if (tail && k0 + n * 8 + e >= lim[i]) x = -INFINITY;
              top = fmaxf(top, x);
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * p.scale_log2;
          // The maximum moves only when this block's P would pass 2^15.
          const bool need = top > mx[i] + 15.0f;
          if (__any_sync(0xffffffffu, need)) {
            const float f = need ? ex2_approx(mx[i] - (top - kHeadroom)) : 1.0f;
            if (need) mx[i] = top - kHeadroom;
            sum[i] *= f;
#pragma unroll
            for (int n = 0; n < D / 8; n++) {
              o[n][2 * i] *= f;
              o[n][2 * i + 1] *= f;
            }
          }
          const float sub = mx[i] == -INFINITY ? 0.0f : mx[i];  // no key so far: all P are 0
          float part = 0.0f;
#pragma unroll
          for (int n = 0; n < C::KEYS / 8; n++) {
            const float x0 = ex2_approx(fmaf(s[n][2 * i], p.scale_log2, -sub));
            const float x1 = ex2_approx(fmaf(s[n][2 * i + 1], p.scale_log2, -sub));
            part += x0 + x1;
            pf[n >> 1][(n & 1) * 2 + i] = pack16x2<T>(x0, x1);
          }
          sum[i] += part;
        }
        wait(&full[vslot], (used + 1) / C::NST);
#pragma unroll
        for (int h = 0; h < C::KEYS / 16; h++) {
          // Values behind the last key may be anything: they count as 0.
          uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
          if (cut) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int k = k0 + h * 16 + i * 8;
              keep[i] = k + 1 < sg.nk ? 0xffffffffu : k < sg.nk ? 0xffffu : 0u;
            }
          }
#pragma unroll
          for (int n2 = 0; n2 < D / 16; n2++) {
            uint32_t b[4];
            ldmatrix4_trans(b, ring + vslot * C::TILE_BYTES + (vrow + h * 16) * 128 +
                                   (n2 >> 2) * C::CHUNK_BYTES +
                                   ((((n2 & 3) * 2 + vpiece) ^ (vrow & 7)) << 4));
            if (cut) {
              b[0] &= keep[0];
              b[1] &= keep[1];
              b[2] &= keep[0];
              b[3] &= keep[1];
            }
            mma_16816<T>(o[2 * n2], pf[h], b[0], b[1]);
            mma_16816<T>(o[2 * n2 + 1], pf[h], b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) {
        if (idle) mbar_arrive(&empty[kslot]);
        mbar_arrive(&empty[vslot]);
      }
      used += 2;
    }
    // --------------------------------------------------------- the pair's result
#pragma unroll
    for (int i = 0; i < 2; i++) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    }
    const bool whole = b0 == 0 && cnt == sg.blocks;
    float *part = p.parts + (long long)(2 * cta + (b0 > 0 ? 0 : 1)) * C::PART;
    // Columns col .. of row r: to the output, or to this CTA's part.
    auto put = [&](int r, int col, const auto &acc, float top, float l) {
      if (whole) {
        finish_row<D, OutT>(p, sg, r, col, acc, top, l);
      } else {
        *reinterpret_cast<std::decay_t<decltype(acc)> *>(part + r * D + col) = acc;
        if (col == 0) reinterpret_cast<float2 *>(part + C::ROWS * D)[r] = make_float2(top, l);
      }
    };
#pragma unroll
    for (int i = 0; i < 2; i++)
      if ((lane & 3) == 0) ml[warp * 16 + qa + i * 8] = make_float2(mx[i], sum[i]);
    named_barrier(1, 32 * C::WARPS);
    // Each share's O is brought to the rows' common maximum.
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int rr = qa + i * 8;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < C::KW; w++) top = fmaxf(top, ml[(rw * C::KW + w) * 16 + rr].x);
      const float f = mx[i] == -INFINITY ? 0.0f : ex2_approx(mx[i] - top);
      float *row = merge + (warp * 16 + rr) * D;
      if (rw * 16 + rr < nrows) {
#pragma unroll
        for (int n = 0; n < D / 8; n++)
          *reinterpret_cast<float2 *>(row + ((n * 8 + qc) ^ (qa << 3))) =
              make_float2(o[n][2 * i] * f, o[n][2 * i + 1] * f);
      }
    }
    named_barrier(1, 32 * C::WARPS);
    for (int x = tid; x < nrows * (D / 4); x += 32 * C::WARPS) {
      const int r = x / (D / 4), col = (x - r * (D / 4)) * 4;
      const int w0 = (r >> 4) * C::KW, rr = r & 15;
      float top = -INFINITY, l = 0.0f;
#pragma unroll
      for (int w = 0; w < C::KW; w++) top = fmaxf(top, ml[(w0 + w) * 16 + rr].x);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < C::KW; w++) {
        const float2 e = ml[(w0 + w) * 16 + rr];
        l += e.x == -INFINITY ? e.y : e.y * ex2_approx(e.x - top);  // (its sum is 0, or NaN)
        const float4 v = *reinterpret_cast<const float4 *>(merge + ((w0 + w) * 16 + rr) * D +
                                                           (col ^ ((rr & 7) << 3)));
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
      }
      put(r, col, acc, top, l);
    }
    named_barrier(1, 32 * C::WARPS);  // merge and ml may be written again
    if (b0 == 0 && !whole && tid == 0) {
      const long long end = range_begin(line, ctas, cta) + sg.at + kPairBlocks + sg.blocks - 1;
      p.joins[cta] = DecodeJoin{range_owner(line, ctas, end), sg.row0, sg.nq, sg.kvh};
    }
  } while (advance());
  if (tid == 0 && *abort_flag) atomicOr(rp.err, kErrTimeout);
}

// Joins the parts of the pairs that cuts fell into: a warp per row, its lanes
// the row's columns, eight parts asked for before any is used. (Joined by the
// CTA that finishes last instead, 32 rows of one request over 32768 keys took
// 62 us, with this launch 37; 64 decodes 88.3 us and 87.2.)
template <int D, int RW, typename OutT>
__global__ void __launch_bounds__(128) fa_decode_join_kernel(const __grid_constant__ DecodeParams p) {
  using C = DecodeCfg<D, RW>;
  constexpr int E = D / 32, U = 8;
  typedef typename std::conditional<E == 4, float4, float2>::type Vec;
  pdl_launch_dependents();
  griddep_wait();
  const int first = blockIdx.x, r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const DecodeJoin join = p.joins[first];
  if (join.last < 0 || r >= join.nq * p.group) return;
  // Part x of the pair: O [ROWS][D], then (max, sum) [ROWS].
  auto part = [&](int x) {
    return p.parts + (long long)(2 * (first + x) + (x == 0 ? 1 : 0)) * C::PART;
  };
  auto part_ml = [&](int x) { return reinterpret_cast<const float2 *>(part(x) + C::ROWS * D)[r]; };
  const int parts = join.last - first + 1;
  float top = -INFINITY, l = 0.0f;
  float acc[E] = {};
  for (int x = lane; x < parts; x += 32) top = fmaxf(top, part_ml(x).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  for (int x0 = 0; x0 < parts; x0 += 32) {
    // This lane's part's weight, for all lanes.
    const float2 e = x0 + lane < parts ? part_ml(x0 + lane) : make_float2(-INFINITY, 0.0f);
    const float w = e.x == -INFINITY ? 0.0f : ex2_approx(e.x - top);
    l += w * e.y;
    const int n = min(32, parts - x0);
    for (int x = 0; x < n; x += U) {
      Vec v[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        v[u] = *(reinterpret_cast<const Vec *>(part(x0 + min(x + u, n - 1)) + r * D) + lane);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const float f = x + u < n ? __shfl_sync(0xffffffffu, w, (x + u) & 31) : 0.0f;
#pragma unroll
        for (int i = 0; i < E; i++)
          if (f != 0.0f) acc[i] = fmaf(elem(v[u], i), f, acc[i]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  DecodeSeg sg = {};  // (more than one block of keys, few rows: each sees some)
  sg.row0 = join.row0;
  sg.kvh = join.kvh;
  finish_row<D, OutT>(p, sg, r, lane * E, *reinterpret_cast<const Vec *>(acc), top, l);
}

}  // namespace llmr
