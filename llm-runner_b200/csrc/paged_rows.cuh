// What the causal and paged attention kernels share: the call's parameters,
// where a request's rows are, tensor maps.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ctx.cuh"
#include "prologue.cuh"
#include "ptx.cuh"

namespace llmr {

// Two fp32 values rounded to a word of T; lo lands in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack16x2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16x2<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack16x2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }

// What both attention operators are given. paged: K and V rows are found
// through the block table; otherwise they are packed like the queries.
struct RowsParams {
  int n, tokens, H, Hk, page, num_pages, max_pages, max_q;
  bool paged;
  const int *cu, *kv_lens, *table;
  long long table_stride;
  const void *q, *k, *v;
  void *o;
  float *lse;
  long long qs[2], os[2];        // {row, head}
  long long ks[3], vs[3];        // {page, row, head}
  float scale;
  int *err;
};

// A request's rows from its offsets and length, checked; false (and the error
// bit) if they are out of range.
__device__ __forceinline__ bool check_rows(const RowsParams &p, int begin, int end, int keys, int &row0, int &nq,
                                           int &nk) {
  const bool in = 0 <= begin && begin <= end && end <= p.tokens;
  row0 = begin;
  nq = in ? end - begin : 0;
  nk = p.paged ? keys : nq;
  const bool ok = in && nk >= 0 &&
                  (!p.paged || (nk <= (long long)p.max_pages * p.page && nq <= p.max_q));
  if (!ok) atomicOr(p.err, kErrInput);
  return ok;
}
__device__ __forceinline__ bool request_rows(const RowsParams &p, int r, int &row0, int &nq,
                                             int &nk) {
  return check_rows(p, p.cu[r], p.cu[r + 1], p.paged ? p.kv_lens[r] : 0, row0, nq, nk);
}

// Softmax numerators are taken relative to 2^-kHeadroom times the maximum that
// was current when they began: the largest is 2^kHeadroom then, and fp16 keeps
// its 11 bits down to 2^-(14 + kHeadroom) of it. The maximum moves, and O and the
// sum are rescaled, when a score would pass 2^15, the most an fp16 P may hold.
constexpr float kHeadroom = 6.0f;

// The few-rows kernel's launch and the workspace of its parts (paged_decode.cu).
int launch_decode_any(llmr_ctx *ctx, int D, int rows, llmr_dtype dt, llmr_dtype od, const RowsParams &r,
                      float *parts);
size_t decode_parts_bytes(int rows, int D);

// 16-bit tensor map with 128-byte swizzle; strides in elements, box[0] = 64.
// The element type only names the zeros outside.
inline int make_map16(llmr_ctx *ctx, CUtensorMap *map, const void *base, const long long (&dims)[4],
               const long long (&strides)[3], int box1, int box2) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return fail(ctx, LLMR_ECUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t d[4], st[3];
  for (int i = 0; i < 4; i++) d[i] = (cuuint64_t)dims[i];
  for (int i = 0; i < 3; i++) st[i] = (cuuint64_t)strides[i] * 2;
  cuuint32_t box[4] = {64, (cuuint32_t)box1, (cuuint32_t)box2, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base), d, st, box,
                   estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ctx, LLMR_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return LLMR_OK;
}

// Whether some offset is out of range or order, which is reported: one warp looks
// at all of them, eight at a time.
__device__ __forceinline__ bool check_requests(const RowsParams &p, int lane) {
  bool bad = false;
  for (int r0 = lane; r0 < p.n; r0 += 256) {
    int a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int r = min(r0 + i * 32, p.n - 1);
      a[i] = p.cu[r];
      b[i] = p.cu[r + 1];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) bad |= a[i] < 0 || a[i] > b[i] || b[i] > p.tokens;
  }
  if (bad) atomicOr(p.err, kErrInput);
  return __any_sync(0xffffffffu, bad);
}

}  // namespace llmr
