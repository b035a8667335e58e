// The page planner and the norm + RoPE + cache-write prologue of the paged
// operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ctx.cuh"
#include "prologue.cuh"
#include "ptx.cuh"

namespace llmr {

// ------------------------------------------------------------------ planner
// Request i lacks need_i = ceil((c + n) / P) - ceil(c / P) pages; exclusive
// prefixes of n and need over the requests give every token and every fresh
// page its place, so tokens and pages are then written independently of one
// another: page x of the step (request order) is free_pages[n_free - 1 - x].
// Latency is all that counts (a decode step moves a few KB: 256 requests 4.0 us
// of device time, 48 prompts of 96k tokens 8.6 us, issue on 8 SMs), so it is one
// launch: a cluster of 1 to 8 CTAs, each of which scans all requests itself
// (cheaper than handing the prefixes over) and writes its share of the tokens
// and pages. All reads of arrays that may be written in place come before the
// cluster barrier, all writes after it.
constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxSeqs = 4096;  // 12 bytes of shared memory each

struct PlanParams {
  int n, max_tokens, page, log_page, num_pages, free_cap, max_pages;
  long long table_stride;
  const int *ctx_lens, *new_lens, *free_pages, *n_free;
  int *table, *cu_q, *kv_lens, *positions, *slots, *n_free_out;
  int *err;
};

// Largest i in [0, n) with a[i] <= x, for ascending a with a[0] <= x. Entries
// that are equal (empty ranges) are passed over.
__device__ __forceinline__ int last_at_most(const int *a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive sums over the block of two values at a time, in 64 bits: lengths
// that do not belong there must not wrap into range.
__device__ __forceinline__ void block_scan2(long long &a, long long &b, long long (*part)[2],
                                            int warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    part[warp][0] = a;
    part[warp][1] = b;
  }
  __syncthreads();
  if (warp == 0) {
    long long x = lane < warps ? part[lane][0] : 0, y = lane < warps ? part[lane][1] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += u;
        y += v;
      }
    }
    part[lane][0] = x;
    part[lane][1] = y;
  }
  __syncthreads();
  if (warp > 0) {
    a += part[warp - 1][0];
    b += part[warp - 1][1];
  }
}

// Positions and slots of this thread's places, U neighbouring ones at a time:
// one search, then a walk; the U table loads are asked for together, and
// stored 16 bytes wide where the arrays allow it. Returns whether a page is
// out of range. (One place at a time with divisions by the page size, a step
// of 96k tokens took 12.8 us, all of it issue.)
template <int U>
__device__ __forceinline__ bool plan_places(const PlanParams &p, const int *tok0, const int *page0,
                                            const int *ctx, int free_n, int total, int first, int step) {
  const bool wide =
      U == 4 && ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
  bool odd = false;
  for (long long x0 = (long long)first * U; x0 < p.max_tokens; x0 += (long long)U * step) {
    int pos[U], slot[U], r = x0 < total ? last_at_most(tok0, p.n, (int)x0) : 0;
    const int *from[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int x = (int)x0 + u;
      pos[u] = 0;
      from[u] = nullptr;
      if (x < total) {
        while (x >= tok0[r + 1]) r++;
        pos[u] = ctx[r] + x - tok0[r];
        const int held = (ctx[r] + p.page - 1) >> p.log_page, col = pos[u] >> p.log_page;
        // A fresh page is read where it came from: its table entry may be
        // written by another CTA.
        from[u] = col < held ? p.table + (long long)r * p.table_stride + col
                             : p.free_pages + (free_n - 1 - (page0[r] + col - held));
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) slot[u] = from[u] ? *from[u] : -1;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool in = (unsigned)slot[u] < (unsigned)p.num_pages;
      odd |= from[u] && !in;
      slot[u] = in ? (slot[u] << p.log_page) + (pos[u] & (p.page - 1)) : -1;
    }
    if (wide && x0 + U <= p.max_tokens) {
      *reinterpret_cast<int4 *>(p.positions + x0) = make_int4(pos[0], pos[1 % U], pos[2 % U], pos[3 % U]);
      *reinterpret_cast<int4 *>(p.slots + x0) = make_int4(slot[0], slot[1 % U], slot[2 % U], slot[3 % U]);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++)
        if (x0 + u < p.max_tokens) {
          p.positions[x0 + u] = pos[u];
          p.slots[x0 + u] = slot[u];
        }
    }
  }
  return odd;
}

__global__ void __launch_bounds__(kPlanThreads, 1) paged_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int *tok0 = plan_smem;            // [n + 1] first new token of each request
  int *page0 = tok0 + p.n + 1;      // [n + 1] first fresh page of each request
  int *ctx = page0 + p.n + 1;       // [n]
  __shared__ long long part[32][2];
  const int tid = threadIdx.x, rank = blockIdx.x, ranks = gridDim.x;
  const int warps = blockDim.x >> 5;
  pdl_launch_dependents();
  griddep_wait();
  const int free_n = *p.n_free;
  long long base_t = 0, base_p = 0;
  bool bad = false;
  for (int i0 = 0; i0 < p.n; i0 += blockDim.x) {
    const int i = i0 + tid;
    long long c = 0, t = 0, need = 0;
    if (i < p.n) {
      c = p.ctx_lens[i];
      t = p.new_lens[i];
      if (c < 0 || t < 0 || c + t > (long long)p.max_pages * p.page) {
        bad = true;
        c = t = 0;
      }
      need = ((c + t + p.page - 1) >> p.log_page) - ((c + p.page - 1) >> p.log_page);
    }
    long long a = t, b = need;
    block_scan2(a, b, part, warps);
    // Sums past int are refused below; the prefixes are not used then.
    if (i < p.n) {
      tok0[i] = (int)(base_t + a - t);
      page0[i] = (int)(base_p + b - need);
      ctx[i] = (int)c;
    }
    base_t += part[warps - 1][0];
    base_p += part[warps - 1][1];
    __syncthreads();
  }
  bad = __syncthreads_or(bad) || free_n < 0 || free_n > p.free_cap || base_t > p.max_tokens;
  const bool dry = !bad && base_p > free_n;
  if (tid == 0) {
    tok0[p.n] = (int)base_t;
    page0[p.n] = (int)base_p;
  }
  // (also makes tok0 / page0 visible to the whole block)
  cluster_sync();
  const int step = ranks * blockDim.x, first = rank * blockDim.x + tid;
  if (bad || dry) {
    for (int i = first; i <= p.n; i += step) p.cu_q[i] = 0;
    if (p.kv_lens != p.ctx_lens)
      for (int i = first; i < p.n; i += step) p.kv_lens[i] = p.ctx_lens[i];
    for (int x = first; x < p.max_tokens; x += step) {
      p.positions[x] = 0;
      p.slots[x] = -1;
    }
    if (first == 0) {
      *p.n_free_out = free_n;
      atomicOr(p.err, bad ? kErrInput : kErrPages);
    }
    return;
  }
  const int total_t = (int)base_t, total_p = (int)base_p;
  for (int i = first; i <= p.n; i += step) p.cu_q[i] = tok0[i];
  for (int i = first; i < p.n; i += step) p.kv_lens[i] = ctx[i] + tok0[i + 1] - tok0[i];
  if (first == 0) *p.n_free_out = free_n - total_p;
  for (int x = first; x < total_p; x += step) {
    const int r = last_at_most(page0, p.n, x);
    const int col = ((ctx[r] + p.page - 1) >> p.log_page) + x - page0[r];
    p.table[(long long)r * p.table_stride + col] = p.free_pages[free_n - 1 - x];
  }
  bool odd = p.max_tokens > 4 * step
                 ? plan_places<4>(p, tok0, page0, ctx, free_n, total_t, first, step)
                 : plan_places<1>(p, tok0, page0, ctx, free_n, total_t, first, step);
  if (odd) atomicOr(p.err, kErrInput);
}

// ----------------------------------------------------------------- prologue
// One pass over the new tokens' rows: read, RMSNorm and rotation in fp32
// registers, one rounding, write. Bound by loads in flight. A group of D / 16 lanes holds
// a row as 8 elements of its first half and the 8 elements D/2 further on, so
// that both pairings of the rotation, (2i, 2i+1) and (i, i + D/2), stay inside
// a lane and every access is 16 bytes. A warp takes kRopeSteps rows per
// group of ONE token, all loads issued before the first use. Small CTAs leave a
// choice of register limits: 28 warps per SM at 72 registers. 8191 tokens, 32 / 8
// heads of 128: 46 us, 4.5 TB/s; of 64: 23 us; 2000 tokens of 128: 10.9. 32 warps at
// 64 registers (spills at heads of 64): 45, 24 and 12.1 us; 24 warps at 80: 49.5, 24.3
// and 11.2; in CTAs of 256 threads 49 and 26 at 8191. From fp32 (4 bytes of spill at
// 72 registers) 48.8, 26.6 and 11.7 us = 6.2 TB/s; 24 warps, no spill: 50.2, 26.9, 11.5. Rows per group in CTAs of 256, 8191 tokens of 128: 4 took 64 us (two
// CTAs per SM), 1 took 55 (six).
constexpr int kRopeSteps = 2;
constexpr int kRopeThreads = 64, kRopeCtas = 14;  // CTAs per SM

struct PagedRopeParams {
  int tokens, hq, hk, page, num_pages, rope_rows, chunks;  // chunks: warps per token
  float eps;
  const void *q, *k, *v;
  void *q_out, *k_cache, *v_cache;
  long long qs[2], ks[2], vs[2], os[2];  // {row, head}
  long long kc[3], vc[3];                // {page, row, head}
  const int *positions, *slots;
  const float *q_gain, *k_gain, *cos_t, *sin_t;
  int *err;
};

template <typename T>
__device__ __forceinline__ void load8(float *x, const T *src) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int c = 0; c < 8; c += V) {
    const Pack<T, V> pk = *reinterpret_cast<const Pack<T, V> *>(src + c);
#pragma unroll
    for (int e = 0; e < V; e++) x[c + e] = to_f32<T>(pk.v[e]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *dst, const float *x) {
  Pack<T, 8> pk;
#pragma unroll
  for (int e = 0; e < 8; e++) pk.v[e] = from_f32<T>(x[e]);
  *reinterpret_cast<Pack<T, 8> *>(dst) = pk;
}

template <int D, typename InT, typename OutT, bool HALF>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas)
paged_prologue_kernel(const PagedRopeParams p) {
  constexpr int LANES = D / 16, GROUPS = 32 / LANES;
  const int lane = threadIdx.x & 31;
  const int sub = lane % LANES, grp = lane / LANES;
  const long long item = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
  const int t = (int)(item / p.chunks);
  pdl_launch_dependents();
  griddep_wait();
  if (t >= p.tokens) return;
  const int h0 = (int)(item - (long long)t * p.chunks) * (GROUPS * kRopeSteps);
  // The slot, the position and the rows are asked for together: a token's
  // chain is two loads long (its table row comes second).
  const int slot = p.slots[t];
  const int pos = p.cos_t ? p.positions[t] : 0;
  const int first = p.q ? 0 : p.hq;  // rows: hq of Q, hk of K, hk of V
  const int rows = p.hq + 2 * p.hk;
  float x[kRopeSteps][16] = {};
#pragma unroll
  for (int s = 0; s < kRopeSteps; s++) {
    const int r = first + h0 + s * GROUPS + grp;
    if (r < rows) {
      const InT *src;
      if (r < p.hq)
        src = static_cast<const InT *>(p.q) + t * p.qs[0] + r * p.qs[1];
      else if (r < p.hq + p.hk)
        src = static_cast<const InT *>(p.k) + t * p.ks[0] + (r - p.hq) * p.ks[1];
      else
        src = static_cast<const InT *>(p.v) + t * p.vs[0] + (r - p.hq - p.hk) * p.vs[1];
      load8<InT>(x[s], src + sub * 8);
      load8<InT>(x[s] + 8, src + D / 2 + sub * 8);
    }
  }
  if (slot < 0) return;  // padding
  const int pg = slot / p.page, prow = slot - pg * p.page;
  if (pg >= p.num_pages || pos < 0 || (p.cos_t && pos >= p.rope_rows)) {
    if (lane == 0) atomicOr(p.err, kErrInput);
    return;
  }
  // The token's table row, in the order this lane's elements use it: pair
  // (i, i + D/2) is element i of both halves; pairs (2i, 2i+1) are 4 of the
  // first half and 4 of the second.
  float cv[8], sv[8];
  if (p.cos_t) {
    const float *ct = p.cos_t + (long long)pos * (D / 2), *st = p.sin_t + (long long)pos * (D / 2);
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int at = HALF ? sub * 8 + c * 4 : c * (D / 4) + sub * 4;
      const float4 a = *reinterpret_cast<const float4 *>(ct + at);
      const float4 b = *reinterpret_cast<const float4 *>(st + at);
      cv[4 * c] = a.x; cv[4 * c + 1] = a.y; cv[4 * c + 2] = a.z; cv[4 * c + 3] = a.w;
      sv[4 * c] = b.x; sv[4 * c + 1] = b.y; sv[4 * c + 2] = b.z; sv[4 * c + 3] = b.w;
    }
  }
#pragma unroll
  for (int s = 0; s < kRopeSteps; s++) {
    const int r = first + h0 + s * GROUPS + grp;
    const int kind = r < p.hq ? 0 : r < p.hq + p.hk ? 1 : 2;
    const float *gain = kind == 0 ? p.q_gain : kind == 1 ? p.k_gain : nullptr;
    float *y = x[s];
    if (p.q_gain || p.k_gain) {  // whole warps take part in the sums
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; e++) ss = fmaf(y[e], y[e], ss);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (gain != nullptr) {
        const float rms = rsqrtf(ss / (float)D + p.eps);
        float g[16];
        load8<float>(g, gain + sub * 8);
        load8<float>(g + 8, gain + D / 2 + sub * 8);
#pragma unroll
        for (int e = 0; e < 16; e++) y[e] = y[e] * rms * g[e];
      }
    }
    if (r >= rows) continue;
    if (p.cos_t && kind < 2) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int i0 = HALF ? e : 2 * e, i1 = HALF ? e + 8 : 2 * e + 1;
        const float a = y[i0], b = y[i1];
        y[i0] = a * cv[e] - b * sv[e];
        y[i1] = a * sv[e] + b * cv[e];
      }
    }
    OutT *dst;
    if (kind == 0)
      dst = static_cast<OutT *>(p.q_out) + t * p.os[0] + r * p.os[1];
    else if (kind == 1)
      dst = static_cast<OutT *>(p.k_cache) + pg * p.kc[0] + prow * p.kc[1] + (r - p.hq) * p.kc[2];
    else
      dst = static_cast<OutT *>(p.v_cache) + pg * p.vc[0] + prow * p.vc[1] +
            (r - p.hq - p.hk) * p.vc[2];
    store8<OutT>(dst + sub * 8, y);
    store8<OutT>(dst + D / 2 + sub * 8, y + 8);
  }
}

}  // namespace llmr
