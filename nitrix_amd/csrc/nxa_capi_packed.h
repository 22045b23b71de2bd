// C entry points of packed-sequence attention (part of nxa_capi.hip).
#pragma once

#include "nxa_packed.h"

namespace {

// Head dim 0 < n <= 256 in whole 16-byte chunks.
int check_head_dim(const char* name, int n, int epc) {
  if (n <= 0) return fail(NXA_E_SHAPE, "head dim %s=%d must be positive", name, n);
  if (n > kMaxHeadDim)
    return fail(NXA_E_UNSUPPORTED, "head dim %s=%d exceeds %d", name, n, kMaxHeadDim);
  if (n % epc != 0)
    return fail(NXA_E_UNSUPPORTED, "head dim %s=%d must be a multiple of %d", name, n, epc);
  return NXA_OK;
}

// Strides in whole 16-byte chunks (the last, of rows, bounded for 32-bit
// offsets inside a tile).
int check_strides(const char* name, const int64_t* s, int n, int es) {
  const int epc = 16 / es;
  for (int i = 0; i < n; ++i) {
    if (s[i] < 0) return fail(NXA_E_LAYOUT, "%s stride %d is negative", name, i);
    if (s[i] % epc != 0)
      return fail(NXA_E_LAYOUT, "%s stride %d (%lld) must be a multiple of %d elements", name, i,
                  (long long)s[i], epc);
  }
  if (!row_stride_ok(s[n - 1], es))
    return fail(NXA_E_LAYOUT, "%s row stride %lld: 64 rows must span less than 2^32 bytes", name,
                (long long)s[n - 1]);
  return NXA_OK;
}

int check_ptr16(const char* name, const void* p) {
  if (!p) return fail(NXA_E_ARG, "%s is NULL", name);
  if ((uintptr_t)p % 16) return fail(NXA_E_LAYOUT, "%s must be 16-byte aligned", name);
  return NXA_OK;
}

int check_packed(const nxa_packed_desc* d) {
  if (!d) return fail(NXA_E_ARG, "descriptor is NULL");
  if (!known_dtype(d->io_dtype))
    return fail(NXA_E_DTYPE, "io_dtype %d is not NXA_BF16, NXA_F16 or NXA_F32", d->io_dtype);
  if (d->T <= 0 || d->nseq <= 0 || d->H <= 0 || d->Hk <= 0)
    return fail(NXA_E_SHAPE, "extents must be positive (T=%d nseq=%d H=%d Hk=%d)", d->T, d->nseq,
                d->H, d->Hk);
  if (d->H % d->Hk != 0)
    return fail(NXA_E_SHAPE, "H=%d must be a multiple of Hk=%d", d->H, d->Hk);
  const int es = esize(d->io_dtype);
  int rc = check_head_dim("D", d->D, 16 / es);
  if (!rc) rc = check_head_dim("Dv", d->Dv, 16 / es);
  if (!rc) rc = check_strides("q", d->q_str, 2, es);
  if (!rc) rc = check_strides("k", d->k_str, 2, es);
  if (!rc) rc = check_strides("v", d->v_str, 2, es);
  if (!rc) rc = check_strides("o", d->o_str, 2, es);
  return rc;
}

void set_strides(int64_t (&dst)[3], const int64_t* src) {
  dst[0] = 0;
  dst[1] = src[0];
  dst[2] = src[1];
}

nxa::PackedParams packed_params(const nxa_packed_desc* d, const void* q, const void* k,
                                const void* v, const int32_t* offsets, const void* o,
                                const float* lse) {
  nxa::PackedParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = const_cast<void*>(o);
  p.lse = const_cast<float*>(lse);
  p.offsets = offsets;
  p.nseq = d->nseq;
  p.T = d->T;
  p.Hk = d->Hk;
  p.G = d->H / d->Hk;
  p.B = 1;
  p.H = d->H;
  p.Lq = p.Lk = d->T;
  p.D = d->D;
  p.Dv = d->Dv;
  p.causal = d->causal ? 1 : 0;
  p.scale = d->scale;
  p.scale_log2 = d->scale * nxa::kLog2e;
  set_strides(p.q_str, d->q_str);
  set_strides(p.k_str, d->k_str);
  set_strides(p.v_str, d->v_str);
  set_strides(p.o_str, d->o_str);
  return p;
}

int packed_dp(const nxa_packed_desc* d) {
  const int m = d->D > d->Dv ? d->D : d->Dv;
  return m <= 64 ? 64 : m <= 128 ? 128 : 256;
}

int check_packed_grid(const nxa_packed_desc* d, bool bwd) {
  nxa::PackedParams p = packed_params(d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  p.parts = nxa::packed_parts(p);
  const int64_t threads = bwd ? nxa::packed_bwd_threads(p, d->io_dtype, packed_dp(d))
                              : nxa::packed_fwd_threads(p, d->io_dtype, packed_dp(d));
  if (threads >= (int64_t)1 << 32)
    return fail(NXA_E_SHAPE, "H=%d T=%d nseq=%d exceed a grid of 2^32 threads", d->H, d->T, d->nseq);
  return NXA_OK;
}

}  // namespace

extern "C" {

int nxa_packed_check(const nxa_packed_desc* desc) {
  const int rc = check_packed(desc);
  return rc ? rc : check_packed_grid(desc, false);
}

int nxa_packed_fwd(const nxa_packed_desc* d, const void* q, const void* k, const void* v,
                   const int32_t* offsets, void* o, void* o_lo, float* lse, void* stream) {
  int rc = nxa_packed_check(d);
  if (!rc) rc = check_ptr16("q", q);
  if (!rc) rc = check_ptr16("k", k);
  if (!rc) rc = check_ptr16("v", v);
  if (!rc) rc = check_ptr16("o", o);
  if (rc) return rc;
  if (!offsets) return fail(NXA_E_ARG, "offsets is NULL");
  if (o_lo && (uintptr_t)o_lo % 16) return fail(NXA_E_LAYOUT, "o_lo must be 16-byte aligned");
  nxa::PackedParams p = packed_params(d, q, k, v, offsets, o, lse);
  p.o_lo = d->io_dtype == NXA_F32 ? nullptr : o_lo;
  hipStream_t s = (hipStream_t)stream;
  return launch("packed_fwd", s, [&] { nxa::launch_packed_fwd(p, d->io_dtype, packed_dp(d), s); });
}

size_t nxa_packed_workspace_bytes(const nxa_packed_desc* d) {
  if (check_packed(d) || check_packed_grid(d, true)) return 0;
  const nxa::PackedParams p = packed_params(d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  return 2 * align256((size_t)d->H * d->T * 4) + 4 * nxa::packed_part_floats(p);
}

int nxa_packed_bwd(const nxa_packed_desc* d, const void* q, const void* k, const void* v,
                   const int32_t* offsets, const void* o, const void* o_lo, const float* lse,
                   const void* dout,
                   const int64_t* do_str, void* dq, const int64_t* dq_str, void* dk,
                   const int64_t* dk_str, void* dv, const int64_t* dv_str, void* workspace,
                   size_t workspace_bytes, void* stream) {
  int rc = check_packed(d);
  if (!rc) rc = check_packed_grid(d, true);
  const void* ptrs[8] = {q, k, v, o, dout, dq, dk, dv};
  const char* names[8] = {"q", "k", "v", "o", "dout", "dq", "dk", "dv"};
  for (int i = 0; i < 8 && !rc; ++i) rc = check_ptr16(names[i], ptrs[i]);
  if (rc) return rc;
  if (!offsets || !lse || !do_str || !dq_str || !dk_str || !dv_str)
    return fail(NXA_E_ARG, "offsets, lse and the strides must not be NULL");
  const int es = esize(d->io_dtype);
  if (!rc) rc = check_strides("dout", do_str, 2, es);
  if (!rc) rc = check_strides("dq", dq_str, 2, es);
  if (!rc) rc = check_strides("dk", dk_str, 2, es);
  if (!rc) rc = check_strides("dv", dv_str, 2, es);
  if (rc) return rc;
  const size_t need = nxa_packed_workspace_bytes(d);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
    return fail(NXA_E_WORKSPACE, "workspace of %zu bytes, %zu needed (256-byte aligned)",
                workspace ? workspace_bytes : (size_t)0, need);
  if (o_lo && (uintptr_t)o_lo % 16) return fail(NXA_E_LAYOUT, "o_lo must be 16-byte aligned");
  nxa::PackedParams p = packed_params(d, q, k, v, offsets, o, lse);
  p.o_lo = d->io_dtype == NXA_F32 ? nullptr : const_cast<void*>(o_lo);
  p.dout = dout;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  set_strides(p.do_str, do_str);
  set_strides(p.dq_str, dq_str);
  set_strides(p.dk_str, dk_str);
  set_strides(p.dv_str, dv_str);
  const size_t rows = align256((size_t)d->H * d->T * 4);
  p.nlse2 = (float*)workspace;
  p.ndelta = (float*)((char*)workspace + rows);
  p.parts = nxa::packed_parts(p);
  p.dkv_part = (float*)((char*)workspace + 2 * rows);
  hipStream_t s = (hipStream_t)stream;
  return launch("packed_bwd", s, [&] { nxa::launch_packed_bwd(p, d->io_dtype, packed_dp(d), s); });
}

}  // extern "C"
