// C entry points of the paged key-value cache (part of nxa_capi.hip).
#pragma once

#include "nxa_paged.h"
#include "nxa_pages.h"

namespace {

// (page and slot numbers plus what a block steps by stay in 31 bits)
constexpr int kMostPages = 1 << 30;
// (a grid holds less than 2^32 threads: 256 for four tokens written, 256 a listed row)
constexpr int kMostTokens = (1 << 26) - 4, kMostListed = 1 << 24;

int check_pool(const nxa_pool_desc* d) {
  if (!d) return fail(NXA_E_ARG, "pool descriptor is NULL");
  if (!known_dtype(d->io_dtype))
    return fail(NXA_E_DTYPE, "io_dtype %d is not NXA_BF16, NXA_F16 or NXA_F32", d->io_dtype);
  if (d->P <= 0 || d->Hk <= 0 || d->PS <= 0)
    return fail(NXA_E_SHAPE, "extents must be positive (P=%d Hk=%d PS=%d)", d->P, d->Hk, d->PS);
  if (d->P > kMostPages || d->PS > kMostPages)
    return fail(NXA_E_SHAPE, "P=%d, PS=%d: at most 2^30 pages of 2^30 tokens", d->P, d->PS);
  const int es = esize(d->io_dtype);
  int rc = check_head_dim("D", d->D, 16 / es);
  if (!rc) rc = check_head_dim("Dv", d->Dv, 16 / es);
  if (!rc) rc = check_strides("k_pages", d->k_str, 3, es);
  if (!rc) rc = check_strides("v_pages", d->v_str, 3, es);
  return rc;
}

int check_pool_ptrs(const void* k, const void* v) {
  const int rc = check_ptr16("k_pages", k);
  return rc ? rc : check_ptr16("v_pages", v);
}

void set_pool(nxa::PoolParams& p, const nxa_pool_desc* d, const void* k, const void* v) {
  p.k = const_cast<void*>(k);
  p.v = const_cast<void*>(v);
  for (int i = 0; i < 3; ++i) {
    p.k_str[i] = d->k_str[i];
    p.v_str[i] = d->v_str[i];
  }
  p.P = d->P;
  p.Hk = d->Hk;
  p.PS = d->PS;
  p.D = d->D;
  p.Dv = d->Dv;
}

// A page table of B rows of M entries.
int check_table(int64_t B, int64_t M, int64_t table_rs) {
  if (B <= 0 || M <= 0)
    return fail(NXA_E_SHAPE, "page table extents must be positive (B=%lld M=%lld)", (long long)B,
                (long long)M);
  if (table_rs < 0) return fail(NXA_E_LAYOUT, "page table row stride is negative");
  return NXA_OK;
}

struct PagedPlan {
  int strips, nblk;
};

int plan_paged(int Hk, int PS, int Dv, int B, int M, int H, bool (*whole)(int64_t, int64_t),
               int most, int start, PagedPlan* plan) {
  if (H <= 0 || H % Hk != 0)
    return fail(NXA_E_SHAPE, "H=%d must be a positive multiple of Hk=%d", H, Hk);
  // (zeros of a sequence without tokens are counted in 31 bits, 256 at a time)
  if ((int64_t)H * Dv > ((int64_t)1 << 31) - 256)
    return fail(NXA_E_SHAPE, "H=%d heads of %d: more than 2^31 - 256 elements a sequence", H, Dv);
  plan->strips = (H / Hk + 15) / 16;
  // Units of the largest table, in 31 bits a head.
  const int64_t room = (int64_t)M * PS;
  const int64_t len = room < INT32_MAX ? room : INT32_MAX;
  const int64_t tiles = (int64_t)B * ((len + nxa::kPagedKeys - 1) / nxa::kPagedKeys + start);
  const int64_t rows = (int64_t)B * Hk * plan->strips;
  if (tiles >= (int64_t)1 << 31 || rows >= (int64_t)1 << 31)
    return fail(NXA_E_SHAPE, "%d sequences of up to %lld tokens exceed 2^31 tiles", B,
                (long long)len);
  // (a block a row where a grid of less than 2^32 threads holds them)
  const int64_t units = tiles * Hk * plan->strips;
  plan->nblk = whole(room, rows) && rows < 1 << 24 ? 0 : (int)(units < most ? units : most);
  return NXA_OK;
}

int plan_paged(const nxa_pool_desc* d, int B, int M, int H, PagedPlan* plan) {
  return plan_paged(
      d->Hk, d->PS, d->Dv, B, M, H, [](int64_t room, int64_t) { return nxa::paged_whole(room); },
      nxa::kPagedBlocks, nxa::kStartUnits, plan);
}

size_t paged_workspace(int dp, const PagedPlan& plan) {
  return (size_t)plan.nblk * (2 * nxa::paged_part_floats(dp) * 4 + sizeof(int4));
}

size_t paged_workspace(const nxa_pool_desc* d, const PagedPlan& plan) {
  return paged_workspace(nxa::paged_dp(d->D > d->Dv ? d->D : d->Dv), plan);
}

// Free, extend and fork: contiguous tables, results in arrays of their own.
int check_rows(int B, int M, int P, int PS, const void* table, const void* lengths,
               const void* refs, const void* table_out, const void* lengths_out,
               const void* refs_out) {
  if (B <= 0 || M <= 0 || P <= 0 || PS <= 0)
    return fail(NXA_E_SHAPE, "extents must be positive (B=%d M=%d P=%d PS=%d)", B, M, P, PS);
  if (P > kMostPages || B > kMostPages)
    return fail(NXA_E_SHAPE, "B=%d, P=%d: at most 2^30 rows and pages", B, P);
  if ((int64_t)M * PS >= (int64_t)1 << 31)
    return fail(NXA_E_SHAPE, "a row of %d pages of %d tokens has room for 2^31 or more", M, PS);
  if (!table || !lengths || !refs || !table_out || !lengths_out || !refs_out)
    return fail(NXA_E_ARG, "a table, lengths or refs pointer is NULL");
  if (table == table_out || lengths == lengths_out || refs == refs_out)
    return fail(NXA_E_ARG, "results need arrays of their own");
  return NXA_OK;
}

nxa::RowsParams rows_params(int B, int M, int P, int PS, const int32_t* table,
                            const int32_t* lengths, const int32_t* refs, int32_t* table_out,
                            int32_t* lengths_out, int32_t* refs_out) {
  nxa::RowsParams p = {};
  p.table = table;
  p.lengths = lengths;
  p.refs = refs;
  p.table_out = table_out;
  p.lengths_out = lengths_out;
  p.refs_out = refs_out;
  p.B = B;
  p.M = M;
  p.P = P;
  p.PS = PS;
  return p;
}

int need_workspace(const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need || (uintptr_t)ws % 16))
    return fail(NXA_E_WORKSPACE, "workspace of %zu bytes, %zu needed (16-byte aligned)",
                ws ? have : (size_t)0, need);
  return NXA_OK;
}

size_t fork_workspace(int B, int P, int n) {
  if (B <= 0 || P <= 0 || n < 0) return 0;
  return ((size_t)n + B + (n < P ? n : P)) * 4;
}

size_t compact_workspace(int P) {
  if (P <= 0 || P > kMostPages) return 0;
  const size_t nb = ((size_t)P + nxa::kCompactPages - 1) / nxa::kCompactPages;
  return (nb + 4 + 3 * (size_t)P) * 4;
}

// Copies, forks and compaction of a checked pool: PoolParams, es its elements'
// bytes, or QuantPool, es its scales'.
template <typename Pool>
int pages_copy(const char* name, const Pool& p, int es, const int32_t* src, const int32_t* dst,
               int n, void* stream) {
  if (n < 0 || (n > 0 && (!src || !dst))) return fail(NXA_E_ARG, "n=%d pairs", n);
  if ((int64_t)(n < nxa::kCopyPairs ? n : nxa::kCopyPairs) * p.Hk * 256 >= (int64_t)1 << 32)
    return fail(NXA_E_SHAPE, "Hk=%d exceeds the grid", p.Hk);
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= p.P || dst[i] < 0 || dst[i] >= p.P)
      return fail(NXA_E_ARG, "pair %d (%d -> %d) is outside the pool's %d pages", i, src[i],
                  dst[i], p.P);
  hipStream_t s = (hipStream_t)stream;
  return launch(name, s, [&] {
    nxa::CopyPairs c;
    for (int i = 0; i < n; i += c.n) {
      c.n = n - i < nxa::kCopyPairs ? n - i : nxa::kCopyPairs;
      memcpy(c.src, src + i, c.n * sizeof(int));
      memcpy(c.dst, dst + i, c.n * sizeof(int));
      nxa::launch_pages_copy(p, es, c, s);
    }
  });
}

template <typename Pool>
int pages_fork(const char* name, const Pool& pool, int es, int B, int M, const int32_t* table,
               const int32_t* lengths, const int32_t* refs, const int32_t* src,
               const int32_t* dst, int n, int32_t* table_out, int32_t* lengths_out,
               int32_t* refs_out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc =
      check_rows(B, M, pool.P, pool.PS, table, lengths, refs, table_out, lengths_out, refs_out);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!src || !dst))) return fail(NXA_E_ARG, "n=%d forks", n);
  if (n >= kMostListed) return fail(NXA_E_SHAPE, "n=%d: less than 2^24 forks a call", n);
  if (pool.Hk >= 65535) return fail(NXA_E_SHAPE, "Hk=%d exceeds the grid", pool.Hk);
  rc = need_workspace(workspace, workspace_bytes, n ? fork_workspace(B, pool.P, n) : 0);
  if (rc) return rc;
  nxa::RowsParams p =
      rows_params(B, M, pool.P, pool.PS, table, lengths, refs, table_out, lengths_out, refs_out);
  p.rows = src;
  p.counts = dst;
  p.n = n;
  p.work = (int*)workspace;
  hipStream_t s = (hipStream_t)stream;
  return launch(name, s, [&] { nxa::launch_pages_fork(p, pool, es, s); });
}

template <typename Pool>
int pages_compact(const char* name, const Pool& pool, int es, int64_t entries,
                  const int32_t* table, const int32_t* refs, int32_t* table_out,
                  int32_t* refs_out, void* workspace, size_t workspace_bytes, void* stream) {
  if (entries < 0) return fail(NXA_E_SHAPE, "%lld table entries", (long long)entries);
  if ((entries && (!table || !table_out)) || !refs || !refs_out)
    return fail(NXA_E_ARG, "a table or refs pointer is NULL");
  if ((entries && table == table_out) || refs == refs_out)
    return fail(NXA_E_ARG, "results need arrays of their own");
  const int rc = need_workspace(workspace, workspace_bytes, compact_workspace(pool.P));
  if (rc) return rc;
  nxa::CompactParams p = {};
  p.table = table;
  p.refs = refs;
  p.table_out = table_out;
  p.refs_out = refs_out;
  p.entries = entries;
  p.P = pool.P;
  p.Hk = pool.Hk;
  p.PS = pool.PS;
  int* w = (int*)workspace;
  p.movers = w;
  p.holes = w + p.P;
  p.mover_rank = w + 2 * (size_t)p.P;
  p.info = w + 3 * (size_t)p.P;
  p.counts = p.info + 4;
  hipStream_t s = (hipStream_t)stream;
  return launch(name, s, [&] { nxa::launch_pages_compact(p, pool, es, s); });
}

}  // namespace

extern "C" {

int nxa_pool_check(const nxa_pool_desc* desc) { return check_pool(desc); }

size_t nxa_paged_workspace_bytes(const nxa_pool_desc* d, int32_t B, int32_t M, int32_t H) {
  PagedPlan plan;
  if (check_pool(d) || check_table(B, M, 0) || plan_paged(d, B, M, H, &plan)) return 0;
  return paged_workspace(d, plan);
}

int nxa_paged_fwd(const nxa_pool_desc* d, const void* k_pages, const void* v_pages, const void* q,
                  const int64_t* q_str, const int32_t* table, int64_t table_rs,
                  const int32_t* lengths, int32_t B, int32_t M, int32_t H, float scale, void* o,
                  const int64_t* o_str, void* workspace, size_t workspace_bytes, void* stream) {
  PagedPlan plan;
  int rc = check_pool(d);
  if (!rc) rc = check_pool_ptrs(k_pages, v_pages);
  if (!rc) rc = check_ptr16("q", q);
  if (!rc) rc = check_ptr16("o", o);
  if (!rc) rc = check_table(B, M, table_rs);
  if (!rc) rc = plan_paged(d, B, M, H, &plan);
  if (rc) return rc;
  if (!table || !lengths || !q_str || !o_str)
    return fail(NXA_E_ARG, "table, lengths and the strides must not be NULL");
  const int es = esize(d->io_dtype);
  rc = check_strides("q", q_str, 2, es);
  if (!rc) rc = check_strides("o", o_str, 2, es);
  if (!rc) rc = need_workspace(workspace, workspace_bytes, paged_workspace(d, plan));
  if (rc) return rc;
  nxa::PagedParams p = {};
  set_pool(p, d, k_pages, v_pages);
  p.q = q;
  p.o = o;
  for (int i = 0; i < 2; ++i) {
    p.q_str[i] = q_str[i];
    p.o_str[i] = o_str[i];
  }
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
  return launch("paged_fwd", s, [&] { nxa::launch_paged(p, d->io_dtype, s); });
}

int nxa_pages_write(const nxa_pool_desc* d, void* k_pages, void* v_pages, const void* k,
                    const int64_t* k_str, const void* v, const int64_t* v_str, int64_t T,
                    const int32_t* table, int64_t table_rs, const int32_t* starts,
                    const int32_t* offsets, int32_t B, int32_t M, void* stream) {
  int rc = check_pool(d);
  if (!rc) rc = check_pool_ptrs(k_pages, v_pages);
  if (!rc) rc = check_ptr16("k", k);
  if (!rc) rc = check_ptr16("v", v);
  if (!rc) rc = check_table(B, M, table_rs);
  if (rc) return rc;
  if (!table || !starts || !k_str || !v_str)
    return fail(NXA_E_ARG, "table, starts and the strides must not be NULL");
  if (T <= 0 || T > kMostTokens)
    return fail(NXA_E_SHAPE, "T=%lld: 1 to 2^26 - 4 tokens a call", (long long)T);
  if (!offsets && T != B)
    return fail(NXA_E_SHAPE, "without offsets one token a sequence is written: T=%lld, B=%d",
                (long long)T, B);
  rc = check_strides("k", k_str, 2, esize(d->io_dtype));
  if (!rc) rc = check_strides("v", v_str, 2, esize(d->io_dtype));
  if (rc) return rc;
  nxa::WriteParams p = {};
  set_pool(p, d, k_pages, v_pages);
  p.ks = k;
  p.vs = v;
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
  p.es = esize(d->io_dtype);
  hipStream_t s = (hipStream_t)stream;
  return launch("pages_write", s, [&] { nxa::launch_pages_write(p, s); });
}

int nxa_pages_copy(const nxa_pool_desc* d, void* k_pages, void* v_pages, const int32_t* src,
                   const int32_t* dst, int32_t n, void* stream) {
  int rc = check_pool(d);
  if (!rc) rc = check_pool_ptrs(k_pages, v_pages);
  if (rc) return rc;
  nxa::PoolParams p = {};
  set_pool(p, d, k_pages, v_pages);
  return pages_copy("pages_copy", p, esize(d->io_dtype), src, dst, n, stream);
}

int nxa_pages_free(int32_t B, int32_t M, int32_t P, const int32_t* table, const int32_t* lengths,
                   const int32_t* refs, const int32_t* rows, int32_t n, int32_t* table_out,
                   int32_t* lengths_out, int32_t* refs_out, void* stream) {
  const int rc = check_rows(B, M, P, 1, table, lengths, refs, table_out, lengths_out, refs_out);
  if (rc) return rc;
  if (n < 0 || (n > 0 && !rows)) return fail(NXA_E_ARG, "n=%d rows", n);
  if (n >= kMostListed) return fail(NXA_E_SHAPE, "n=%d: less than 2^24 rows a call", n);
  nxa::RowsParams p = rows_params(B, M, P, 1, table, lengths, refs, table_out, lengths_out, refs_out);
  p.rows = rows;
  p.n = n;
  hipStream_t s = (hipStream_t)stream;
  return launch("pages_free", s, [&] { nxa::launch_pages_free(p, s); });
}

int nxa_pages_extend(int32_t B, int32_t M, int32_t P, int32_t PS, const int32_t* table,
                     const int32_t* lengths, const int32_t* refs, const int32_t* counts,
                     int32_t* table_out, int32_t* lengths_out, int32_t* refs_out, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int rc = check_rows(B, M, P, PS, table, lengths, refs, table_out, lengths_out, refs_out);
  if (rc) return rc;
  if (!counts) return fail(NXA_E_ARG, "counts is NULL");
  rc = need_workspace(workspace, workspace_bytes, (size_t)P * 4);
  if (rc) return rc;
  nxa::RowsParams p = rows_params(B, M, P, PS, table, lengths, refs, table_out, lengths_out, refs_out);
  p.counts = counts;
  p.work = (int*)workspace;
  hipStream_t s = (hipStream_t)stream;
  return launch("pages_extend", s, [&] { nxa::launch_pages_extend(p, s); });
}

size_t nxa_pages_fork_workspace_bytes(int32_t B, int32_t P, int32_t n) {
  return fork_workspace(B, P, n);
}

int nxa_pages_fork(const nxa_pool_desc* d, void* k_pages, void* v_pages, int32_t B, int32_t M,
                   const int32_t* table, const int32_t* lengths, const int32_t* refs,
                   const int32_t* src, const int32_t* dst, int32_t n, int32_t* table_out,
                   int32_t* lengths_out, int32_t* refs_out, void* workspace,
                   size_t workspace_bytes, void* stream) {
  int rc = check_pool(d);
  if (!rc) rc = check_pool_ptrs(k_pages, v_pages);
  if (rc) return rc;
  nxa::PoolParams pool = {};
  set_pool(pool, d, k_pages, v_pages);
  return pages_fork("pages_fork", pool, esize(d->io_dtype), B, M, table, lengths, refs, src, dst, n,
                    table_out, lengths_out, refs_out, workspace, workspace_bytes, stream);
}

size_t nxa_pages_compact_workspace_bytes(int32_t P) { return compact_workspace(P); }

int nxa_pages_compact(const nxa_pool_desc* d, void* k_pages, void* v_pages, int64_t entries,
                      const int32_t* table, const int32_t* refs, int32_t* table_out,
                      int32_t* refs_out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_pool(d);
  if (!rc) rc = check_pool_ptrs(k_pages, v_pages);
  if (rc) return rc;
  nxa::PoolParams pool = {};
  set_pool(pool, d, k_pages, v_pages);
  return pages_compact("pages_compact", pool, esize(d->io_dtype), entries, table, refs, table_out,
                       refs_out, workspace, workspace_bytes, stream);
}

}  // extern "C"
