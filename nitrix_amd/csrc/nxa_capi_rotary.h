// C entry points of the rotary positions (part of nxa_capi.hip).
#pragma once

#include "nxa_rotary.h"

namespace {

int check_rotary(const nxa_rotary_desc* d) {
  if (!d) return fail(NXA_E_ARG, "descriptor is NULL");
  if (!known_dtype(d->io_dtype))
    return fail(NXA_E_DTYPE, "io_dtype %d is not NXA_BF16, NXA_F16 or NXA_F32", d->io_dtype);
  if (d->B <= 0 || d->T <= 0 || d->H <= 0 || d->Hk < 0)
    return fail(NXA_E_SHAPE, "extents must be positive (B=%d T=%d H=%d Hk=%d)", d->B, d->T, d->H,
                d->Hk);
  // (a block counts its tokens' elements in 31 bits)
  if ((int64_t)d->H + d->Hk > 1 << 20)
    return fail(NXA_E_SHAPE, "H=%d, Hk=%d: at most 2^20 heads together", d->H, d->Hk);
  if (d->D <= 0 || d->D > nxa::kRotaryMaxDim)
    return fail(NXA_E_UNSUPPORTED, "head dim D=%d is outside 1 .. %d", d->D, nxa::kRotaryMaxDim);
  if (d->R <= 0 || d->R > d->D || d->R % 2)
    return fail(NXA_E_ARG, "R=%d rotated elements: an even number up to D=%d", d->R, d->D);
  if ((int64_t)d->B * (((int64_t)d->T + 3) / 4) >= 1 << 24)
    return fail(NXA_E_SHAPE, "B=%d, T=%d exceed the grid", d->B, d->T);
  for (int i = 0; i < 3; ++i)
    if (d->q_str[i] < 0 || d->k_str[i] < 0 || d->q_out_str[i] < 0 || d->k_out_str[i] < 0)
      return fail(NXA_E_LAYOUT, "stride %d is negative", i);
  if (d->pos_str[0] < 0 || d->pos_str[1] < 0)
    return fail(NXA_E_LAYOUT, "a stride of the positions is negative");
  return NXA_OK;
}

}  // namespace

extern "C" {

int nxa_rotary_check(const nxa_rotary_desc* desc) { return check_rotary(desc); }

int nxa_rotary(const nxa_rotary_desc* d, const void* q, const void* k, const void* positions,
               const double* frequencies, void* q_out, void* k_out, void* stream) {
  const int rc = check_rotary(d);
  if (rc) return rc;
  if (!q || !q_out || (d->Hk > 0 && (!k || !k_out)) || !positions || !frequencies)
    return fail(NXA_E_ARG, "q, k, positions, frequencies and the outputs must not be NULL");
  const size_t es = esize(d->io_dtype);
  if (!aligned(q, es) || !aligned(k, es) || !aligned(q_out, es) || !aligned(k_out, es))
    return fail(NXA_E_LAYOUT, "a pointer is not aligned to its elements");
  nxa::RotaryParams p = {};
  p.x[0] = q, p.x[1] = k;
  p.y[0] = q_out, p.y[1] = k_out;
  p.H[0] = d->H, p.H[1] = d->Hk;
  // Whole 16-byte chunks, none of which holds turned and copied elements (half
  // layout: nor elements of both halves).
  const int epc = 16 / (int)es;
  bool chunks = d->D % epc == 0 && (d->interleaved ? d->R : d->R / 2) % epc == 0;
  for (int w = 0; w < (d->Hk > 0 ? 2 : 1); ++w) {
    chunks = chunks && aligned(p.x[w], 16) && aligned(p.y[w], 16);
    for (int i = 0; i < 3; ++i) {
      p.x_str[w][i] = w ? d->k_str[i] : d->q_str[i];
      p.y_str[w][i] = w ? d->k_out_str[i] : d->q_out_str[i];
      chunks = chunks && p.x_str[w][i] % epc == 0 && p.y_str[w][i] % epc == 0;
    }
  }
  p.positions = positions;
  p.pos_str[0] = d->pos_str[0], p.pos_str[1] = d->pos_str[1];
  p.freq = frequencies;
  p.B = d->B, p.T = d->T, p.D = d->D, p.R = d->R;
  p.interleaved = d->interleaved != 0;
  p.inverse = d->inverse != 0;
  p.pos64 = d->pos64 != 0;
  p.scale = d->scale;
  hipStream_t s = (hipStream_t)stream;
  return launch("rotary", s, [&] { nxa::launch_rotary(p, d->io_dtype, chunks, s); });
}

}  // extern "C"
