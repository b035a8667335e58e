// Launches of the few-rows paged attention kernel (fa_decode.cuh), in a
// source of their own: its variants take as long to compile as all the rest.
#include "fa_decode.cuh"
#include "kattr.cuh"

namespace llmr {

template <int D, int RW, typename T, typename OutT>
int launch_decode(llmr_ctx *ctx, const RowsParams &r, float *parts) {
  using C = DecodeCfg<D, RW>;
  DecodeParams p;
  p.rows = r;
  p.group = r.H / r.Hk;
  p.scale_log2 = r.scale * 1.4426950408889634f;
  p.parts = parts;
  p.joins = reinterpret_cast<DecodeJoin *>(parts + (size_t)kDecodeCtas * 2 * C::PART);
  CUtensorMap mk, mv;
  int rc;
  if ((rc = make_map16(ctx, &mk, r.k, {D, r.page, r.Hk, r.num_pages}, {r.ks[1], r.ks[2], r.ks[0]},
                       r.page < C::BN ? r.page : C::BN, 1)) ||
      (rc = make_map16(ctx, &mv, r.v, {D, r.page, r.Hk, r.num_pages}, {r.vs[1], r.vs[2], r.vs[0]},
                       r.page < C::BN ? r.page : C::BN, 1)))
    return rc;
  auto kern = fa_decode_kernel<D, RW, T, OutT>;
  CUDA_TRY(ctx, set_smem_once(kern, C::SMEM_BYTES));
  // Two CTAs share an SM only where there is no free one: under a budget, one CTA
  // for each of its SMs.
  const int want = ctx->num_sms < ctx->total_sms ? ctx->num_sms : 2 * ctx->num_sms;
  const int grid = want < kDecodeCtas ? want : kDecodeCtas;
  CUDA_TRY(ctx, launch_overlapped(kern, dim3(grid), C::THREADS, C::SMEM_BYTES, ctx->stream, 1, mk, mv, p));
  if ((rc = after_launch(ctx, "fa_decode"))) return rc;
  CUDA_TRY(ctx, launch_overlapped(fa_decode_join_kernel<D, RW, OutT>, dim3(grid, (r.max_q * p.group + 3) / 4), 128,
                                  0, ctx->stream, 1, p));
  return after_launch(ctx, "fa_decode_join");
}

template <int D, int RW>
int launch_decode_t(llmr_ctx *ctx, llmr_dtype dt, llmr_dtype od, const RowsParams &r, float *parts) {
  if (dt == LLMR_F16) {
    if (od == LLMR_F32) return launch_decode<D, RW, __half, float>(ctx, r, parts);
    if (od == LLMR_F16) return launch_decode<D, RW, __half, __half>(ctx, r, parts);
    return launch_decode<D, RW, __half, __nv_bfloat16>(ctx, r, parts);
  }
  if (od == LLMR_F32) return launch_decode<D, RW, __nv_bfloat16, float>(ctx, r, parts);
  if (od == LLMR_F16) return launch_decode<D, RW, __nv_bfloat16, __half>(ctx, r, parts);
  return launch_decode<D, RW, __nv_bfloat16, __nv_bfloat16>(ctx, r, parts);
}

int launch_decode_any(llmr_ctx *ctx, int D, int rows, llmr_dtype dt, llmr_dtype od, const RowsParams &r,
                      float *parts) {
  if (rows <= 16)
    return D == 128 ? launch_decode_t<128, 1>(ctx, dt, od, r, parts)
                    : launch_decode_t<64, 1>(ctx, dt, od, r, parts);
  return D == 128 ? launch_decode_t<128, 2>(ctx, dt, od, r, parts)
                  : launch_decode_t<64, 2>(ctx, dt, od, r, parts);
}

size_t decode_parts_bytes(int rows, int D) {
  const size_t r = rows <= 16 ? 16 : 32;
  return (size_t)kDecodeCtas * (2 * r * (D + 2) * sizeof(float) + sizeof(DecodeJoin));
}

}  // namespace llmr
