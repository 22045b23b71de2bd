// Quantised paged key-value cache: parameter blocks and launchers of
// nxa_qpages.hip (writing and reading back) and nxa_qpaged.hip (one new token a
// sequence attends its pages).
//
// A row (token and head) of D elements is held as codes of 4 or 8 bits with a
// scale s and a minimum z of the model's type T: s = T((max - min) * float(1 /
// (2^bits - 1))), code = rint((x - z) / s), value = z + s code.  Pools: k codes [P, Hk, PS,
// D bits / 8 bytes], v codes likewise, scales [P, Hk, PS, 4] of T (k's s and z,
// v's s and z); the slots of a page and head lie end to end, so that a step of an
// attention is one run of each.  In 4 bits element 2 i is the low half of byte i.
#pragma once

#include "nxa_paged.h"

namespace nxa {

// A pool of codes: k and v of PoolParams with strides in bytes, and the scales
// with strides in elements.
struct QuantPool : PoolParams {
  void* sc;
  int64_t sc_str[2];  // page, head
  int bits;
};

// Written (ks / vs to the pool) or read back (the pool to ks / vs).
struct QuantMoveParams {
  QuantPool pool;
  void *ks, *vs;                 // [Hk, T, D], [Hk, T, Dv]
  int64_t ks_str[2], vs_str[2];  // head, token
  const int* offsets;            // [B + 1], or null: token s is sequence s's
  const int* starts;             // [B]
  const int* table;
  int64_t table_rs;
  int64_t T;
  int B, M;
};

struct QuantPagedParams : PagedParams {  // k_str, v_str in bytes
  const void* sc;
  int64_t sc_str[2];
  int bits;
  int k16, v16, s16;  // page strides in 16 bytes (set by the launcher)
};

// What starting on a row costs a block, in units of 128 tokens (its first page ids,
// copies and q, with nothing to work on meanwhile).  us a call with 1 / 3 / 5 / 8: 64
// sequences of up to 8192 tokens, 4 bits, 61 / 54 / 54 / 56, 8 bits 88 / 73 / 73 / 78; two
// of up to 400000 135 / 134 / 130 / 129.
constexpr int kQuantStart = 5;
int qpaged_dp(int m);  // padded head dim
bool qpaged_whole(int64_t room, int64_t rows);  // a block a row (sequence and head)
int qpaged_blocks(int io_dtype, int dp, int bits);  // most blocks that share the work

void launch_quant_write(const QuantMoveParams& p, int io_dtype, hipStream_t stream);
void launch_quant_read(const QuantMoveParams& p, int io_dtype, hipStream_t stream);
void launch_quant_paged(const QuantPagedParams& p, int io_dtype, hipStream_t stream);

}  // namespace nxa
