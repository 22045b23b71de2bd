// C entry points of the quantised paged cache (part of nxa_capi.hip, after
// nxa_capi_paged.h).
#pragma once

#include "nxa_quant.h"

namespace {

int check_quant_pool(const nxa_quant_pool_desc* d) {
  if (!d) return fail(NXA_E_ARG, "pool descriptor is NULL");
  if (!known_dtype(d->io_dtype))
    return fail(NXA_E_DTYPE, "io_dtype %d is not NXA_BF16, NXA_F16 or NXA_F32", d->io_dtype);
  if (d->bits != 4 && d->bits != 8)
    return fail(NXA_E_UNSUPPORTED, "codes of %d bits: 4 or 8", d->bits);
  if (d->P <= 0 || d->Hk <= 0 || d->PS <= 0)
    return fail(NXA_E_SHAPE, "extents must be positive (P=%d Hk=%d PS=%d)", d->P, d->Hk, d->PS);
  if (d->P > kMostPages || d->PS > kMostPages)
    return fail(NXA_E_SHAPE, "P=%d, PS=%d: at most 2^30 pages of 2^30 tokens", d->P, d->PS);
  if (d->Hk > 1 << 24) return fail(NXA_E_SHAPE, "Hk=%d: at most 2^24 heads", d->Hk);
  int rc = check_head_dim("D", d->D, 8);
  if (!rc) rc = check_head_dim("Dv", d->Dv, 8);
  if (rc) return rc;
  for (int i = 0; i < 2; ++i) {
    if (d->k_str[i] < 0 || d->v_str[i] < 0 || d->s_str[i] < 0)
      return fail(NXA_E_LAYOUT, "pool stride %d is negative", i);
    if (d->k_str[i] % 4 || d->v_str[i] % 4 || d->s_str[i] % 4)
      return fail(NXA_E_LAYOUT, "pool stride %d must be a multiple of 4", i);
  }
  return NXA_OK;
}

int check_quant_ptrs(const void* k, const void* v, const void* scales) {
  int rc = check_ptr16("k_pages", k);
  if (!rc) rc = check_ptr16("v_pages", v);
  return rc ? rc : check_ptr16("scales", scales);
}

void set_quant_pool(nxa::QuantPool& p, const nxa_quant_pool_desc* d, const void* k, const void* v,
                    const void* scales) {
  p.k = const_cast<void*>(k);
  p.v = const_cast<void*>(v);
  p.sc = const_cast<void*>(scales);
  for (int i = 0; i < 2; ++i) {
    p.k_str[i] = d->k_str[i];
    p.v_str[i] = d->v_str[i];
    p.sc_str[i] = d->s_str[i];
  }
  p.P = d->P;
  p.Hk = d->Hk;
  p.PS = d->PS;
  p.D = d->D;
  p.Dv = d->Dv;
  p.bits = d->bits;
}

int quant_move(const char* name, bool write, const nxa_quant_pool_desc* d, const void* k_pages,
               const void* v_pages, const void* scales, const void* k, const int64_t* k_str,
               const void* v, const int64_t* v_str, int64_t T, const int32_t* table,
               int64_t table_rs, const int32_t* starts, const int32_t* offsets, int32_t B,
               int32_t M, void* stream) {
  int rc = check_quant_pool(d);
  if (!rc) rc = check_quant_ptrs(k_pages, v_pages, scales);
  if (!rc) rc = check_ptr16("k", k);
  if (!rc) rc = check_ptr16("v", v);
  if (!rc) rc = check_table(B, M, table_rs);
  if (rc) return rc;
  if (!table || !starts || !k_str || !v_str)
    return fail(NXA_E_ARG, "table, starts and the strides must not be NULL");
  if (T <= 0 || T > kMostTokens)
    return fail(NXA_E_SHAPE, "T=%lld: 1 to 2^26 - 4 tokens a call", (long long)T);
  if (!offsets && T != B)
    return fail(NXA_E_SHAPE, "without offsets there is one token a sequence: T=%lld, B=%d",
                (long long)T, B);
  rc = check_strides("k", k_str, 2, esize(d->io_dtype));
  if (!rc) rc = check_strides("v", v_str, 2, esize(d->io_dtype));
  if (rc) return rc;
  nxa::QuantMoveParams p = {};
  set_quant_pool(p.pool, d, k_pages, v_pages, scales);
  p.ks = const_cast<void*>(k);
  p.vs = const_cast<void*>(v);
  for (int i = 0; i < 2; ++i) {
    p.ks_str[i] = k_str[i];
    p.vs_str[i] = v_str[i];
  }
  p.offsets = offsets;
  p.starts = starts;
  p.table = table;
  p.table_rs = table_rs;
  p.T = T;
  p.B = B;
  p.M = M;
  hipStream_t s = (hipStream_t)stream;
  return launch(name, s, [&] {
    if (write) nxa::launch_quant_write(p, d->io_dtype, s);
    else nxa::launch_quant_read(p, d->io_dtype, s);
  });
}

int plan_quant_paged(const nxa_quant_pool_desc* d, int B, int M, int H, PagedPlan* plan) {
  // (a wave steps past a row's last token: what it adds stays in 31 bits)
  if ((int64_t)M * d->PS >= ((int64_t)1 << 31) - 4096)
    return fail(NXA_E_SHAPE, "a row of %d pages of %d tokens has room for 2^31 or more", M, d->PS);
  const int most = nxa::qpaged_blocks(d->io_dtype, nxa::qpaged_dp(d->D > d->Dv ? d->D : d->Dv),
                                      d->bits);
  return plan_paged(d->Hk, d->PS, d->Dv, B, M, H, nxa::qpaged_whole, most, nxa::kQuantStart,
                    plan);
}

size_t quant_paged_workspace(const nxa_quant_pool_desc* d, const PagedPlan& plan) {
  return paged_workspace(nxa::qpaged_dp(d->D > d->Dv ? d->D : d->Dv), plan);
}

}  // namespace

extern "C" {

int nxa_quant_pool_check(const nxa_quant_pool_desc* desc) { return check_quant_pool(desc); }

int nxa_quant_write(const nxa_quant_pool_desc* d, void* k_pages, void* v_pages, void* scales,
                    const void* k, const int64_t* k_str, const void* v, const int64_t* v_str,
                    int64_t T, const int32_t* table, int64_t table_rs, const int32_t* starts,
                    const int32_t* offsets, int32_t B, int32_t M, void* stream) {
  return quant_move("quant_write", true, d, k_pages, v_pages, scales, k, k_str, v, v_str, T, table,
                    table_rs, starts, offsets, B, M, stream);
}

int nxa_quant_read(const nxa_quant_pool_desc* d, const void* k_pages, const void* v_pages,
                   const void* scales, void* k, const int64_t* k_str, void* v,
                   const int64_t* v_str, int64_t T, const int32_t* table, int64_t table_rs,
                   const int32_t* starts, const int32_t* offsets, int32_t B, int32_t M,
                   void* stream) {
  return quant_move("quant_read", false, d, k_pages, v_pages, scales, k, k_str, v, v_str, T, table,
                    table_rs, starts, offsets, B, M, stream);
}

size_t nxa_quant_paged_workspace_bytes(const nxa_quant_pool_desc* d, int32_t B, int32_t M,
                                       int32_t H) {
  PagedPlan plan;
  if (check_quant_pool(d) || check_table(B, M, 0) || plan_quant_paged(d, B, M, H, &plan)) return 0;
  return quant_paged_workspace(d, plan);
}

int nxa_quant_paged_fwd(const nxa_quant_pool_desc* d, const void* k_pages, const void* v_pages,
                        const void* scales, const void* q, const int64_t* q_str,
                        const int32_t* table, int64_t table_rs, const int32_t* lengths, int32_t B,
                        int32_t M, int32_t H, float scale, void* o, const int64_t* o_str,
                        void* workspace, size_t workspace_bytes, void* stream) {
  PagedPlan plan;
  int rc = check_quant_pool(d);
  if (!rc) rc = check_quant_ptrs(k_pages, v_pages, scales);
  if (!rc) rc = check_ptr16("q", q);
  if (!rc) rc = check_ptr16("o", o);
  if (!rc) rc = check_table(B, M, table_rs);
  if (!rc) rc = plan_quant_paged(d, B, M, H, &plan);
  if (rc) return rc;
  if (!table || !lengths || !q_str || !o_str)
    return fail(NXA_E_ARG, "table, lengths and the strides must not be NULL");
  const int es = esize(d->io_dtype);
  rc = check_strides("q", q_str, 2, es);
  if (!rc) rc = check_strides("o", o_str, 2, es);
  if (!rc) rc = need_workspace(workspace, workspace_bytes, quant_paged_workspace(d, plan));
  if (rc) return rc;
  nxa::QuantPool pool = {};
  set_quant_pool(pool, d, k_pages, v_pages, scales);
  nxa::QuantPagedParams p = {};
  static_cast<nxa::PoolParams&>(p) = pool;
  p.sc = scales;
  p.bits = d->bits;
  for (int i = 0; i < 2; ++i) {
    p.sc_str[i] = d->s_str[i];
    p.q_str[i] = q_str[i];
    p.o_str[i] = o_str[i];
  }
  p.q = q;
  p.o = o;
  p.table = table;
  p.lengths = lengths;
  p.table_rs = table_rs;
  p.B = B;
  p.M = M;
  p.G = H / d->Hk;
  p.strips = plan.strips;
  p.nblk = plan.nblk;
  p.scale_log2 = scale * nxa::kLog2e;
  p.joins = (int4*)workspace;
  p.part = (float*)(p.joins + plan.nblk);
  hipStream_t s = (hipStream_t)stream;
  return launch("quant_paged_fwd", s, [&] { nxa::launch_quant_paged(p, d->io_dtype, s); });
}

int nxa_quant_copy(const nxa_quant_pool_desc* d, void* k_pages, void* v_pages, void* scales,
                   const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  int rc = check_quant_pool(d);
  if (!rc) rc = check_quant_ptrs(k_pages, v_pages, scales);
  if (rc) return rc;
  nxa::QuantPool p = {};
  set_quant_pool(p, d, k_pages, v_pages, scales);
  return pages_copy("quant_copy", p, esize(d->io_dtype), src, dst, n, stream);
}

int nxa_quant_fork(const nxa_quant_pool_desc* d, void* k_pages, void* v_pages, void* scales,
                   int32_t B, int32_t M, const int32_t* table, const int32_t* lengths,
                   const int32_t* refs, const int32_t* src, const int32_t* dst, int32_t n,
                   int32_t* table_out, int32_t* lengths_out, int32_t* refs_out, void* workspace,
                   size_t workspace_bytes, void* stream) {
  int rc = check_quant_pool(d);
  if (!rc) rc = check_quant_ptrs(k_pages, v_pages, scales);
  if (rc) return rc;
  nxa::QuantPool p = {};
  set_quant_pool(p, d, k_pages, v_pages, scales);
  return pages_fork("quant_fork", p, esize(d->io_dtype), B, M, table, lengths, refs, src, dst, n,
                    table_out, lengths_out, refs_out, workspace, workspace_bytes, stream);
}

int nxa_quant_compact(const nxa_quant_pool_desc* d, void* k_pages, void* v_pages, void* scales,
                      int64_t entries, const int32_t* table, const int32_t* refs,
                      int32_t* table_out, int32_t* refs_out, void* workspace,
                      size_t workspace_bytes, void* stream) {
  int rc = check_quant_pool(d);
  if (!rc) rc = check_quant_ptrs(k_pages, v_pages, scales);
  if (rc) return rc;
  nxa::QuantPool p = {};
  set_quant_pool(p, d, k_pages, v_pages, scales);
  return pages_compact("quant_compact", p, esize(d->io_dtype), entries, table, refs, table_out,
                       refs_out, workspace, workspace_bytes, stream);
}

}  // extern "C"
