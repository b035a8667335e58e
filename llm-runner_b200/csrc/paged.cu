// Host side of the causal and paged operators of include/llmr_attn.h:
// argument checks, tensor maps, the choice of kernel and the launches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <string.h>

#include "ctx.cuh"
#include "fa_rows.cuh"
#include "kattr.cuh"
#include "paged_kernels.cuh"

using namespace llmr;

namespace {

// Makes the context's device current for one call and puts the caller's back.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (cudaGetDevice(&old_) != cudaSuccess) old_ = device;
    ok_ = old_ == device || cudaSetDevice(device) == cudaSuccess;
    changed_ = old_ != device;
  }
  ~OnDevice() {
    if (changed_) cudaSetDevice(old_);
  }
  bool ok() const { return ok_; }

 private:
  int old_ = 0;
  bool ok_ = false, changed_ = false;
};

// An exception (the host is out of memory) ends as a status at the C boundary,
// with a message where there is memory for one.
int out_of_memory(llmr_ctx *ctx) {
  try {
    return fail(ctx, LLMR_ENOMEM, "the host is out of memory");
  } catch (...) {
    if (ctx) ctx->err.clear();  // not an older call's
    return LLMR_ENOMEM;
  }
}
#define NO_THROW_BEGIN try {
#define NO_THROW_END(ctx)      \
  }                            \
  catch (...) {                \
    return out_of_memory(ctx); \
  }
#define ENTER(ctx)                                   \
  if (!(ctx)) return LLMR_EINVAL;                    \
  OnDevice on_device_((ctx)->device);                \
  if (!on_device_.ok()) return fail(ctx, LLMR_ECUDA, "cudaSetDevice(%d) failed", (ctx)->device)

bool is16(llmr_dtype t) { return t == LLMR_F16 || t == LLMR_BF16; }
bool known(llmr_dtype t) { return t == LLMR_F32 || is16(t); }
size_t size_of(llmr_dtype t) { return t == LLMR_F32 ? 4 : 2; }
bool a16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool a4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
long long either(uint64_t given, long long dense) { return given ? (long long)given : dense; }
// Strides that are whole 16-byte pieces and below the 2^40 bytes a tensor
// map can hold.
bool strides16(std::initializer_list<long long> st, size_t es) {
  for (long long s : st)
    if (s < 0 || s >= (1ll << 40) / (long long)es || (s * (long long)es) % 16) return false;
  return true;
}

// What is wrong with the head geometry, or null.
const char *bad_heads(uint32_t H, uint32_t Hk, uint32_t D) {
  if (D != 64 && D != 128) return "head_dim must be 64 or 128";
  if (H < 1 || Hk < 1 || H > 65535 || H % Hk) return "n_heads must be a multiple of n_kv_heads";
  if (H / Hk > 128) return "more than 128 query heads per key/value head";
  return nullptr;
}

const char *bad_page(uint32_t page, uint32_t num_pages) {
  if (page != 16 && page != 32 && page != 64 && page != 128 && page != 256)
    return "page_size must be 16, 32, 64, 128 or 256";
  if (num_pages < 1 || (uint64_t)num_pages * page > 0x7fffffffull)
    return "num_pages must be at least 1 and num_pages * page_size below 2^31";
  return nullptr;
}

const char *bad_paged(const llmr_paged_desc *d) {
  if (const char *e = bad_heads(d->n_heads, d->n_kv_heads, d->head_dim)) return e;
  if (const char *e = bad_page(d->page_size, d->num_pages)) return e;
  if (!is16(d->dtype) || !known(d->out_dtype)) return "q and the caches must be fp16 or bf16";
  if (!(d->scale > 0.0f) || !isfinite(d->scale)) return "scale must be finite and > 0";
  if (d->n_seqs > 0x3fffffffu || d->total_tokens > 0x3fffffffu) return "problem too large";
  // (A length rounded up to a block of keys, and the end of its last block, are ints.)
  if (d->max_pages < 1 || (uint64_t)d->max_pages * d->page_size > 0x7fffff00ull)
    return "max_pages must be at least 1 and max_pages * page_size at most 2^31 - 256";
  if (d->table_stride && d->table_stride < d->max_pages) return "table_stride is below max_pages";
  return nullptr;
}

// Workspace of the paged chunk kernel: two parts per CTA (O, maximum and sum of
// 256 rows) and its unit to join.
size_t chunk_parts_bytes(int D) {
  return (size_t)kMaxRanges * (2 * 256 * (D + 2) * sizeof(float) + sizeof(FaJoin));
}

template <int D, typename T, typename OutT, bool PAGED>
int launch_fa_rows(llmr_ctx *ctx, const RowsParams &r) {
  using C = FaRowsCfg<D>;
  FaRowsParams p = {};
  p.rows = r;
  p.group = r.H / r.Hk;
  p.tpt = 128 / p.group;
  p.tu = 2 * p.tpt;
  p.recip = (65536 + p.group - 1) / p.group;
  p.scale_log2 = r.scale * 1.4426950408889634f;
  int grid;
  if (PAGED) {
    grid = ctx->num_sms < kMaxRanges ? ctx->num_sms : kMaxRanges;
    p.part_o = static_cast<float *>(ctx->ws);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + (size_t)2 * kMaxRanges * 256 * D);
    p.joins = reinterpret_cast<FaJoin *>(p.part_ml + (size_t)2 * kMaxRanges * 256);
  } else {
    // Fewer units than SMs: units of one tile, whose keys both softmax groups
    // share, so that a unit takes half as long and there are twice as many.
    // 1500 tokens, 14 / 2 heads of 64: 17.0 us instead of 25.1; 700 tokens, 32 / 8
    // heads of 128: 15.5 and 18.9. With more units than SMs reading K and V for
    // one tile mostly costs more than that gains (1500 tokens, 32 / 8 heads of
    // 128: 33.3 us instead of 30.1), but not just above one unit per SM (3000
    // tokens, 14 / 2 heads of 64, 167 units: 37.7 and 43.8).
    if ((long long)r.tokens / (2 * p.tpt) * r.Hk < ctx->total_sms) p.tu = p.tpt;
    const long long vt = (long long)r.tokens / p.tu + r.n, units = vt * r.Hk;
    if (units > 0x7fffffffLL) return fail(ctx, LLMR_EINVAL, "problem too large");
    p.vtiles = (int)vt;
    p.units = (int)units;
    // With an SM budget the grid is that small and strides over the units.
    p.dynamic = units > ctx->num_sms && ctx->num_sms == ctx->total_sms;
    grid = p.dynamic || units < ctx->num_sms ? (int)units : ctx->num_sms;
    p.shares = grid < ctx->num_sms ? grid : ctx->num_sms;
    if (p.shares > kMaxShares) p.shares = kMaxShares;
  }
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = make_map16(ctx, &mq, r.q, {D, p.group, r.tokens, r.Hk},
                       {r.qs[1], r.qs[0], r.qs[1] * p.group}, p.group, p.tpt)))
    return rc;
  auto kv_map = [&](CUtensorMap *m, const void *base, const long long *st) {
    if (PAGED)
      return make_map16(ctx, m, base, {D, r.page, r.Hk, r.num_pages}, {st[1], st[2], st[0]},
                        r.page < 128 ? r.page : 128, 1);
    return make_map16(ctx, m, base, {D, r.tokens, r.Hk, 1}, {st[1], st[2], st[1]}, 128, 1);
  };
  if ((rc = kv_map(&mk, r.k, r.ks)) || (rc = kv_map(&mv, r.v, r.vs))) return rc;
  auto kern = fa_rows_kernel<D, T, OutT, PAGED>;
  CUDA_TRY(ctx, set_smem_once(kern, C::SMEM_BYTES));
  // setmaxnreg.inc waits until the registers it asks for are free within
  // the block's launch allocation: never launch a split that cannot fit.
  int regs = 0;
  CUDA_TRY(ctx, launch_regs(kern, &regs));
  if (regs * C::THREADS < C::REG_NEED)
    return fail(ctx, LLMR_ECUDA, "fa_rows: %d launch registers per thread are too few for the "
                "register split", regs);
  if constexpr (!PAGED) {
    // (Overlapped with the call before, ragged prompts took 9 % longer: CTAs of
    // two grids that both take over units. Grids that do not take over units were
    // not measured overlapped.)
    kern<<<grid, C::THREADS, C::SMEM_BYTES, ctx->stream>>>(mq, mk, mv, p);
    return after_launch(ctx, "fa_rows");
  } else {
    CUDA_TRY(ctx, launch_overlapped(kern, dim3(grid), C::THREADS, C::SMEM_BYTES, ctx->stream, 1, mq, mk, mv, p));
    if ((rc = after_launch(ctx, "fa_rows"))) return rc;
    CUDA_TRY(ctx, launch_overlapped(fa_rows_join_kernel<D, OutT>, dim3(grid, 8), 256, 0, ctx->stream, 1, p));
    return after_launch(ctx, "fa_rows_join");
  }
}

template <int D, typename T, bool PAGED>
int launch_fa_rows_o(llmr_ctx *ctx, llmr_dtype od, const RowsParams &r) {
  if (od == LLMR_F32) return launch_fa_rows<D, T, float, PAGED>(ctx, r);
  if (od == LLMR_F16) return launch_fa_rows<D, T, __half, PAGED>(ctx, r);
  return launch_fa_rows<D, T, __nv_bfloat16, PAGED>(ctx, r);
}

template <bool PAGED>
int launch_fa_rows_any(llmr_ctx *ctx, int D, llmr_dtype dt, llmr_dtype od, const RowsParams &r) {
  if (D == 128)
    return dt == LLMR_F16 ? launch_fa_rows_o<128, __half, PAGED>(ctx, od, r)
                          : launch_fa_rows_o<128, __nv_bfloat16, PAGED>(ctx, od, r);
  return dt == LLMR_F16 ? launch_fa_rows_o<64, __half, PAGED>(ctx, od, r)
                        : launch_fa_rows_o<64, __nv_bfloat16, PAGED>(ctx, od, r);
}

// Query rows per (request, key/value head) up to which the decode kernel runs.
// 32 requests over 4096 keys, 8 key/value heads of 128: 32 rows 95 us there and
// 106 us in fa_rows; one request over 32768: 33.6 and 38.4. (48 rows, in a form
// that held up to 64, took 172 us and 112; one request 98 and 43.)
constexpr uint32_t kDecodeRows = 32;

uint32_t rows_per_head(const llmr_paged_desc *d) {
  const uint64_t q = d->max_q_len < d->total_tokens ? d->max_q_len : d->total_tokens;
  const uint64_t rows = q * (d->n_heads / d->n_kv_heads);
  return rows > 0xffffffffull ? 0xffffffffu : (uint32_t)rows;
}

template <int D, typename InT, typename OutT>
int launch_paged_prologue(llmr_ctx *ctx, bool half, PagedRopeParams &p) {
  constexpr int per_warp = (32 / (D / 16)) * kRopeSteps;
  const int rows = (p.q ? p.hq : 0) + 2 * p.hk;
  p.chunks = (rows + per_warp - 1) / per_warp;
  const long long warps = (long long)p.tokens * p.chunks;
  constexpr int per_cta = kRopeThreads / 32;
  const unsigned grid = (unsigned)((warps + per_cta - 1) / per_cta);
  auto kern = half ? paged_prologue_kernel<D, InT, OutT, true> : paged_prologue_kernel<D, InT, OutT, false>;
  CUDA_TRY(ctx, launch_overlapped(kern, dim3(grid), kRopeThreads, 0, ctx->stream, 1, p));
  return after_launch(ctx, "paged_prologue");
}

template <int D, typename InT>
int launch_paged_prologue_o(llmr_ctx *ctx, llmr_dtype od, bool half, PagedRopeParams &p) {
  return od == LLMR_F16 ? launch_paged_prologue<D, InT, __half>(ctx, half, p)
                        : launch_paged_prologue<D, InT, __nv_bfloat16>(ctx, half, p);
}

}  // namespace

extern "C" {

int llmr_attention_causal(llmr_ctx *ctx, const llmr_causal_desc *d, const int32_t *cu_seqlens,
                          const void *q, const void *k, const void *v, void *o, float *lse) NO_THROW_BEGIN
  ENTER(ctx);
  if (!d) return fail(ctx, LLMR_EINVAL, "null argument");
  if (const char *e = bad_heads(d->n_heads, d->n_kv_heads, d->head_dim))
    return fail(ctx, LLMR_EINVAL, "%s", e);
  if (!is16(d->dtype) || !known(d->out_dtype))
    return fail(ctx, LLMR_EINVAL, "q, k and v must be fp16 or bf16");
  if (!(d->scale > 0.0f) || !isfinite(d->scale))
    return fail(ctx, LLMR_EINVAL, "scale must be finite and > 0");
  if (d->n_seqs > 0x3fffffffu || d->total_tokens > 0x3fffffffu)
    return fail(ctx, LLMR_EINVAL, "problem too large");
  if (d->n_seqs == 0 || d->total_tokens == 0) return LLMR_OK;
  if (!cu_seqlens || !q || !k || !v || !o) return fail(ctx, LLMR_EINVAL, "null argument");
  const long long D = d->head_dim, H = d->n_heads, Hk = d->n_kv_heads;
  RowsParams p = {};
  p.n = (int)d->n_seqs;
  p.tokens = (int)d->total_tokens;
  p.H = (int)H;
  p.Hk = (int)Hk;
  p.page = 1;
  p.num_pages = 1;
  p.cu = cu_seqlens;
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = o;
  p.lse = lse;
  p.qs[0] = either(d->q_row_stride, H * D);
  p.qs[1] = either(d->q_head_stride, D);
  p.ks[1] = either(d->k_row_stride, Hk * D);
  p.ks[2] = either(d->k_head_stride, D);
  p.vs[1] = either(d->v_row_stride, Hk * D);
  p.vs[2] = either(d->v_head_stride, D);
  p.os[0] = either(d->o_row_stride, H * D);
  p.os[1] = either(d->o_head_stride, D);
  p.scale = d->scale;
  p.err = ctx->d_err;
  if (!a16(q) || !a16(k) || !a16(v) || !a16(o) ||
      !strides16({p.qs[0], p.qs[1], p.ks[1], p.ks[2], p.vs[1], p.vs[2]}, 2) ||
      !strides16({p.os[0], p.os[1]}, size_of(d->out_dtype)))
    return fail(ctx, LLMR_EINVAL, "q, k, v, o and their strides must be 16-byte aligned");
  if (!a4(cu_seqlens) || !a4(lse)) return fail(ctx, LLMR_EINVAL, "cu_seqlens or lse is misaligned");
  return launch_fa_rows_any<false>(ctx, (int)D, d->dtype, d->out_dtype, p);
NO_THROW_END(ctx)

size_t llmr_attention_paged_workspace_bytes(const llmr_paged_desc *d) {
  if (!d || bad_paged(d)) return 0;
  if (rows_per_head(d) <= kDecodeRows) return decode_parts_bytes((int)rows_per_head(d), (int)d->head_dim);
  return chunk_parts_bytes((int)d->head_dim);
}

int llmr_attention_paged(llmr_ctx *ctx, const llmr_paged_desc *d, const int32_t *cu_q,
                         const int32_t *kv_lens, const int32_t *block_table, const void *q,
                         const void *k_cache, const void *v_cache, void *o, float *lse) NO_THROW_BEGIN
  ENTER(ctx);
  if (!d) return fail(ctx, LLMR_EINVAL, "null argument");
  if (const char *e = bad_paged(d)) return fail(ctx, LLMR_EINVAL, "%s", e);
  if (d->n_seqs == 0 || d->total_tokens == 0) return LLMR_OK;
  if (d->max_q_len == 0) return fail(ctx, LLMR_EINVAL, "max_q_len must be at least 1");
  if (!cu_q || !kv_lens || !block_table || !q || !k_cache || !v_cache || !o)
    return fail(ctx, LLMR_EINVAL, "null argument");
  const size_t need = llmr_attention_paged_workspace_bytes(d);
  if (need > ctx->ws_bytes)
    return fail(ctx, LLMR_ENOMEM, "workspace %zu bytes < %zu needed (llmr_ctx_reserve)",
                ctx->ws_bytes, need);
  const long long D = d->head_dim, H = d->n_heads, Hk = d->n_kv_heads, P = d->page_size;
  RowsParams p = {};
  p.n = (int)d->n_seqs;
  p.tokens = (int)d->total_tokens;
  p.H = (int)H;
  p.Hk = (int)Hk;
  p.page = (int)P;
  p.num_pages = (int)d->num_pages;
  p.max_pages = (int)d->max_pages;
  p.max_q = (int)(d->max_q_len < d->total_tokens ? d->max_q_len : d->total_tokens);
  p.paged = true;
  p.cu = cu_q;
  p.kv_lens = kv_lens;
  p.table = block_table;
  p.table_stride = either(d->table_stride, d->max_pages);
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.o = o;
  p.lse = lse;
  p.qs[0] = either(d->q_row_stride, H * D);
  p.qs[1] = either(d->q_head_stride, D);
  p.os[0] = either(d->o_row_stride, H * D);
  p.os[1] = either(d->o_head_stride, D);
  p.ks[0] = either(d->k_page_stride, P * Hk * D);
  p.ks[1] = either(d->k_row_stride, Hk * D);
  p.ks[2] = either(d->k_head_stride, D);
  p.vs[0] = either(d->v_page_stride, P * Hk * D);
  p.vs[1] = either(d->v_row_stride, Hk * D);
  p.vs[2] = either(d->v_head_stride, D);
  p.scale = d->scale;
  p.err = ctx->d_err;
  if (!a16(q) || !a16(k_cache) || !a16(v_cache) || !a16(o) ||
      !strides16({p.qs[0], p.qs[1], p.ks[0], p.ks[1], p.ks[2], p.vs[0], p.vs[1], p.vs[2]}, 2) ||
      !strides16({p.os[0], p.os[1]}, size_of(d->out_dtype)))
    return fail(ctx, LLMR_EINVAL, "q, the caches, o and their strides must be 16-byte aligned");
  if (!a4(cu_q) || !a4(kv_lens) || !a4(block_table) || !a4(lse))
    return fail(ctx, LLMR_EINVAL, "cu_q, kv_lens, block_table or lse is misaligned");
  if (rows_per_head(d) <= kDecodeRows) {
    return launch_decode_any(ctx, (int)D, (int)rows_per_head(d), d->dtype, d->out_dtype, p,
                             static_cast<float *>(ctx->ws));
  }
  return launch_fa_rows_any<true>(ctx, (int)D, d->dtype, d->out_dtype, p);
NO_THROW_END(ctx)

int llmr_paged_plan(llmr_ctx *ctx, const llmr_plan_desc *d, const int32_t *ctx_lens,
                    const int32_t *new_lens, const int32_t *free_pages, const int32_t *n_free,
                    int32_t *block_table, int32_t *cu_q, int32_t *kv_lens, int32_t *positions,
                    int32_t *slots, int32_t *n_free_out) NO_THROW_BEGIN
  ENTER(ctx);
  if (!d || !n_free || !cu_q || !n_free_out) return fail(ctx, LLMR_EINVAL, "null argument");
  if (d->n_seqs && (!ctx_lens || !new_lens || !block_table || !kv_lens))
    return fail(ctx, LLMR_EINVAL, "null argument");
  if ((d->free_capacity && !free_pages) || (d->max_tokens && (!positions || !slots)))
    return fail(ctx, LLMR_EINVAL, "null argument");
  if (d->n_seqs > (uint32_t)kPlanMaxSeqs)
    return fail(ctx, LLMR_EINVAL, "n_seqs %u exceeds %d", d->n_seqs, kPlanMaxSeqs);
  if (const char *e = bad_page(d->page_size, d->num_pages)) return fail(ctx, LLMR_EINVAL, "%s", e);
  if (d->max_tokens > 0x3fffffffu || d->free_capacity > 0x3fffffffu ||
      (uint64_t)d->max_pages * d->page_size > 0x7fffffffull)
    return fail(ctx, LLMR_EINVAL, "problem too large");
  if (d->table_stride && d->table_stride < d->max_pages)
    return fail(ctx, LLMR_EINVAL, "table_stride is below max_pages");
  for (const void *x : {(const void *)ctx_lens, (const void *)new_lens, (const void *)free_pages,
                        (const void *)n_free, (const void *)block_table, (const void *)cu_q,
                        (const void *)kv_lens, (const void *)positions, (const void *)slots,
                        (const void *)n_free_out})
    if (!a4(x)) return fail(ctx, LLMR_EINVAL, "an array is misaligned");
  PlanParams p = {};
  p.n = (int)d->n_seqs;
  p.max_tokens = (int)d->max_tokens;
  p.page = (int)d->page_size;
  while ((1 << p.log_page) < p.page) p.log_page++;
  p.num_pages = (int)d->num_pages;
  p.free_cap = (int)d->free_capacity;
  p.max_pages = (int)d->max_pages;
  p.table_stride = either(d->table_stride, d->max_pages);
  p.ctx_lens = ctx_lens;
  p.new_lens = new_lens;
  p.free_pages = free_pages;
  p.n_free = n_free;
  p.table = block_table;
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.positions = positions;
  p.slots = slots;
  p.n_free_out = n_free_out;
  p.err = ctx->d_err;
  // One CTA until there is work for a second round of its threads.
  const long long items = d->max_tokens > d->n_seqs ? d->max_tokens : d->n_seqs;
  const int threads = items <= 256 ? 256 : kPlanThreads;
  int ctas = 1;
  while (ctas < 8 && items > (long long)ctas * threads) ctas *= 2;
  const int smem = (3 * p.n + 2) * (int)sizeof(int);
  CUDA_TRY(ctx, set_smem_once(paged_plan_kernel, (3 * kPlanMaxSeqs + 2) * (int)sizeof(int)));
  CUDA_TRY(ctx, launch_overlapped(paged_plan_kernel, dim3(ctas), threads, smem, ctx->stream, ctas, p));
  return after_launch(ctx, "paged_plan");
NO_THROW_END(ctx)

int llmr_paged_prologue(llmr_ctx *ctx, const llmr_paged_prologue_desc *d,
                        const int32_t *positions, const int32_t *slots, const void *q,
                        const void *k, const void *v, const float *q_gain, const float *k_gain,
                        const float *cos_t, const float *sin_t, void *q_out, void *k_cache,
                        void *v_cache) NO_THROW_BEGIN
  ENTER(ctx);
  if (!d) return fail(ctx, LLMR_EINVAL, "null argument");
  if (const char *e = bad_heads(d->n_heads, d->n_kv_heads, d->head_dim))
    return fail(ctx, LLMR_EINVAL, "%s", e);
  if (const char *e = bad_page(d->page_size, d->num_pages)) return fail(ctx, LLMR_EINVAL, "%s", e);
  if (!known(d->in_dtype) || !is16(d->dtype))
    return fail(ctx, LLMR_EINVAL, "q_out and the caches must be fp16 or bf16");
  if (d->flags & ~(uint32_t)(LLMR_NORM_Q | LLMR_NORM_K | LLMR_ROPE | LLMR_ROPE_HALF))
    return fail(ctx, LLMR_EINVAL, "only NORM_Q, NORM_K, ROPE and ROPE_HALF apply here");
  if ((d->flags & LLMR_ROPE_HALF) && !(d->flags & LLMR_ROPE))
    return fail(ctx, LLMR_EINVAL, "LLMR_ROPE_HALF needs LLMR_ROPE");
  if (d->total_tokens > 0x3fffffffu) return fail(ctx, LLMR_EINVAL, "problem too large");
  if (!isfinite(d->eps) || d->eps < 0.0f) return fail(ctx, LLMR_EINVAL, "eps must be finite and >= 0");
  if (d->total_tokens == 0) return LLMR_OK;
  if (!slots || !k || !v || !k_cache || !v_cache || (q != nullptr) != (q_out != nullptr))
    return fail(ctx, LLMR_EINVAL, "null argument");
  if ((d->flags & LLMR_NORM_Q) && !q_gain) return fail(ctx, LLMR_EINVAL, "LLMR_NORM_Q needs q_gain");
  if ((d->flags & LLMR_NORM_K) && !k_gain) return fail(ctx, LLMR_EINVAL, "LLMR_NORM_K needs k_gain");
  if ((d->flags & LLMR_ROPE) && (!cos_t || !sin_t || !positions || !d->rope_rows))
    return fail(ctx, LLMR_EINVAL, "LLMR_ROPE needs cos/sin tables and positions");
  if (d->rope_rows > 0x7fffffffu) return fail(ctx, LLMR_EINVAL, "problem too large");
  const long long D = d->head_dim, H = d->n_heads, Hk = d->n_kv_heads, P = d->page_size;
  if ((long long)d->total_tokens * (H + 2 * Hk) > (1ll << 33)) return fail(ctx, LLMR_EINVAL, "problem too large");
  PagedRopeParams p = {};
  p.tokens = (int)d->total_tokens;
  p.hq = (int)H;
  p.hk = (int)Hk;
  p.page = (int)P;
  p.num_pages = (int)d->num_pages;
  p.rope_rows = (int)d->rope_rows;
  p.eps = d->eps;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.qs[0] = either(d->q_row_stride, H * D);
  p.qs[1] = either(d->q_head_stride, D);
  p.ks[0] = either(d->k_row_stride, Hk * D);
  p.ks[1] = either(d->k_head_stride, D);
  p.vs[0] = either(d->v_row_stride, Hk * D);
  p.vs[1] = either(d->v_head_stride, D);
  p.os[0] = either(d->q_out_row_stride, H * D);
  p.os[1] = either(d->q_out_head_stride, D);
  p.kc[0] = either(d->k_page_stride, P * Hk * D);
  p.kc[1] = either(d->k_cache_row_stride, Hk * D);
  p.kc[2] = either(d->k_cache_head_stride, D);
  p.vc[0] = either(d->v_page_stride, P * Hk * D);
  p.vc[1] = either(d->v_cache_row_stride, Hk * D);
  p.vc[2] = either(d->v_cache_head_stride, D);
  p.positions = positions;
  p.slots = slots;
  const bool rope = d->flags & LLMR_ROPE;
  p.q_gain = (d->flags & LLMR_NORM_Q) ? q_gain : nullptr;
  p.k_gain = (d->flags & LLMR_NORM_K) ? k_gain : nullptr;
  p.cos_t = rope ? cos_t : nullptr;
  p.sin_t = rope ? sin_t : nullptr;
  p.err = ctx->d_err;
  const size_t es = size_of(d->in_dtype);
  if (!a16(q) || !a16(k) || !a16(v) || !a16(q_out) || !a16(k_cache) || !a16(v_cache) ||
      !a16(p.q_gain) || !a16(p.k_gain) || !a16(p.cos_t) || !a16(p.sin_t) ||
      !strides16({p.qs[0], p.qs[1], p.ks[0], p.ks[1], p.vs[0], p.vs[1]}, es) ||
      !strides16({p.os[0], p.os[1], p.kc[0], p.kc[1], p.kc[2], p.vc[0], p.vc[1], p.vc[2]}, 2))
    return fail(ctx, LLMR_EINVAL, "tensors, gains, tables and strides must be 16-byte aligned");
  if (!a4(positions) || !a4(slots)) return fail(ctx, LLMR_EINVAL, "positions or slots is misaligned");
  if (q != nullptr && q == q_out &&
      (d->in_dtype != d->dtype || p.qs[0] != p.os[0] || p.qs[1] != p.os[1]))
    return fail(ctx, LLMR_EINVAL, "q_out may be q only with its type and strides");
  const bool half = d->flags & LLMR_ROPE_HALF;
#define LLMR_PP(DD)                                                                         \
  return d->in_dtype == LLMR_F32   ? launch_paged_prologue_o<DD, float>(ctx, d->dtype, half, p)   \
         : d->in_dtype == LLMR_F16 ? launch_paged_prologue_o<DD, __half>(ctx, d->dtype, half, p)  \
                                   : launch_paged_prologue_o<DD, __nv_bfloat16>(ctx, d->dtype, half, p)
  if (D == 128) LLMR_PP(128);
  LLMR_PP(64);
#undef LLMR_PP
NO_THROW_END(ctx)

}  // extern "C"
