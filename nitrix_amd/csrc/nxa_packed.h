// Packed sequences: several sequences laid end to end along the token axis,
// sequence s at rows offsets[s] .. offsets[s + 1] - 1, and G query heads to
// each key-value head.  The attention kernels take a PackedParams in place
// of Params; each block finds its (sequence, tile, head) here and then works
// on that sequence as on a dense problem of one head.
//
// A grid needs an upper bound of the tiles without the lengths, which are on
// the device.  Sequence s owns the tile slots from
// S(s) = floor(offsets[s] / TILE) + s on: S grows by at least
// ceil(length / TILE) from one sequence to the next, so every sequence has
// the slots it needs, and there are floor(T / TILE) + (sequences) of them in
// all, at most one a sequence to spare.  S is monotone, so a wave finds the
// sequence of a slot with ballots, 64 probes a step.
//
// Offsets are clamped to 0 .. T and lengths to >= 0 wherever they are read:
// whatever they hold, no block leaves the rows of its tensors.
#pragma once

#include "nxa_common.h"

#include <type_traits>

namespace nxa {

// Strides of the base's q, k, v, o: [1] head, [2] token; Lq = Lk = T.
struct PackedParams : Params {
  const int* offsets;  // nseq + 1
  int nseq, T, Hk, G;
  int slots;           // tile slots of the launching kernel
  int nwork;           // blocks with a slot; those behind zero the unowned rows
  int64_t do_str[3], dq_str[3], dk_str[3], dv_str[3];
};

// What a dK / dV block streams besides its own sequence's base pointers.
struct PackedGroup {
  int heads;                   // query heads of the group
  int64_t q_hs, do_hs, row_hs; // from one head to the next (row_hs: nlse2, ndelta)
  int64_t do_rs, dk_rs, dv_rs; // row strides
};

struct PackedTile {
  int start, len, tile;
};

__device__ __forceinline__ int packed_offset(const PackedParams& pp, int s) {
  return min(max(pp.offsets[s], 0), pp.T);
}

// Sequence and tile of `slot` (all lanes active; uniform results).
__device__ __forceinline__ PackedTile packed_find(const PackedParams& pp, int slot, int tile_rows) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = pp.nseq;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int i = lo + lane * step;
    const bool le = i < hi && packed_offset(pp, i) / tile_rows + i <= slot;
    // (lane 0 always holds: S(lo) <= slot)
    const int cnt = max((int)__popcll(__ballot(le)), 1);
    lo += (cnt - 1) * step;
    hi = min(lo + step, hi);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  PackedTile r;
  r.start = __builtin_amdgcn_readfirstlane(packed_offset(pp, lo));
  r.len = max(__builtin_amdgcn_readfirstlane(packed_offset(pp, lo + 1)) - r.start, 0);
  r.tile = slot - (r.start / tile_rows + lo);
  return r;
}

// Rows outside offsets[0] .. offsets[nseq] of x ([heads][T][n], strides hs,
// rs) become zero; block `blk` of `nblk`.
template <typename T>
__device__ __forceinline__ void packed_zero_rows(const PackedParams& pp, T* x, int heads, int n,
                                                 int64_t hs, int64_t rs, int blk, int nblk) {
  const int lo = packed_offset(pp, 0), hi = max(packed_offset(pp, pp.nseq), lo);
  const int64_t rows = (int64_t)lo + (pp.T - hi);
  const int64_t total = rows * heads * n;
  for (int64_t i = (int64_t)blk * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)nblk * blockDim.x) {
    const int64_t row = i / ((int64_t)heads * n);
    const int rest = (int)(i % ((int64_t)heads * n));
    x[(rest / n) * hs + (row < lo ? row : row - lo + hi) * rs + rest % n] = (T)0.f;
  }
}

// Everything of Params that a packed problem does not have.
__device__ __forceinline__ void packed_base(const PackedParams& pp, Params& p) {
  p = static_cast<const Params&>(pp);
  p.bias = nullptr;
  p.mask = nullptr;
  p.tilemap = nullptr;
  p.order = nullptr;
  p.B = p.H = 1;
  p.has_bias = p.has_mask = p.has_tilemap = 0;
  p.mask_vec = p.bias_vec = 0;
  p.tm_rows = 1;
  p.qk_norm = 0;
  p.qn_on = 0;
  p.dbias_mode = kDbiasNone;
}

// Blocks of the forward and dQ kernels: one query tile of one query head.
// Blocks that run on one XCD (every eighth) take key-value heads x, x + 8, ..
// whole, the query heads that share one after one another, each from its
// last slot (the most keys of a causal tile) down.  False: nothing to do.
template <typename T>
__device__ __forceinline__ bool packed_query_block(const PackedParams& pp, int rows, Params& p,
                                                   int& qt) {
  const int bid = blockIdx.x;
  if (bid >= pp.nwork) {
    // The forward zeroes o, dQ (which runs first of the backward) the three
    // gradients.
    const int blk = bid - pp.nwork, nblk = gridDim.x - pp.nwork;
    if (pp.dq) {
      packed_zero_rows(pp, (T*)pp.dq, pp.Hk * pp.G, pp.D, pp.dq_str[1], pp.dq_str[2], blk, nblk);
      packed_zero_rows(pp, (T*)pp.dk, pp.Hk, pp.D, pp.dk_str[1], pp.dk_str[2], blk, nblk);
      packed_zero_rows(pp, (T*)pp.dv, pp.Hk, pp.Dv, pp.dv_str[1], pp.dv_str[2], blk, nblk);
    } else {
      packed_zero_rows(pp, (T*)pp.o, pp.Hk * pp.G, pp.Dv, pp.o_str[1], pp.o_str[2], blk, nblk);
    }
    return false;
  }
  const int vid = xcd_remap(bid, pp.Hk * pp.G, pp.slots);
  const int hv = vid / pp.slots;
  const int hk = hv % pp.Hk, hq = hk * pp.G + hv / pp.Hk;
  const PackedTile t = packed_find(pp, pp.slots - 1 - vid % pp.slots, rows);
  if ((int64_t)t.tile * rows >= t.len) return false;
  packed_base(pp, p);
  const int64_t r0 = t.start;
  p.q = (const T*)pp.q + hq * pp.q_str[1] + r0 * pp.q_str[2];
  p.k = (const T*)pp.k + hk * pp.k_str[1] + r0 * pp.k_str[2];
  p.v = (const T*)pp.v + hk * pp.v_str[1] + r0 * pp.v_str[2];
  p.o = (T*)pp.o + hq * pp.o_str[1] + r0 * pp.o_str[2];
  const int64_t row = (int64_t)hq * pp.T + r0;
  if (pp.lse) p.lse = pp.lse + row;
  if (pp.dq) {
    p.dout = (const T*)pp.dout + hq * pp.do_str[1] + r0 * pp.do_str[2];
    p.dq = (T*)pp.dq + hq * pp.dq_str[1] + r0 * pp.dq_str[2];
    p.ndelta = pp.ndelta + row;
    p.nlse2 = pp.nlse2 + row;
  }
  p.Lq = p.Lk = t.len;
  qt = t.tile;
  return true;
}

// Blocks of the dK / dV kernels: one key tile of one key-value head, from
// the first slot up (a causal sequence's first keys have the most queries).
template <typename T>
__device__ __forceinline__ bool packed_key_block(const PackedParams& pp, int rows, Params& p,
                                                 int& kt, PackedGroup& grp) {
  const int vid = xcd_remap(blockIdx.x, pp.Hk, pp.slots);
  const int hk = vid / pp.slots;
  const PackedTile t = packed_find(pp, vid % pp.slots, rows);
  if ((int64_t)t.tile * rows >= t.len) return false;
  packed_base(pp, p);
  const int64_t r0 = t.start, hq = (int64_t)hk * pp.G;
  p.q = (const T*)pp.q + hq * pp.q_str[1] + r0 * pp.q_str[2];
  p.k = (const T*)pp.k + hk * pp.k_str[1] + r0 * pp.k_str[2];
  p.v = (const T*)pp.v + hk * pp.v_str[1] + r0 * pp.v_str[2];
  p.dout = (const T*)pp.dout + hq * pp.do_str[1] + r0 * pp.do_str[2];
  p.dk = (T*)pp.dk + hk * pp.dk_str[1] + r0 * pp.dk_str[2];
  p.dv = (T*)pp.dv + hk * pp.dv_str[1] + r0 * pp.dv_str[2];
  p.ndelta = pp.ndelta + hq * pp.T + r0;
  p.nlse2 = pp.nlse2 + hq * pp.T + r0;
  p.Lq = p.Lk = t.len;
  grp.heads = pp.G;
  grp.q_hs = pp.q_str[1], grp.do_hs = pp.do_str[1], grp.row_hs = pp.T;
  grp.do_rs = pp.do_str[2], grp.dk_rs = pp.dk_str[2], grp.dv_rs = pp.dv_str[2];
  kt = t.tile;
  return true;
}

// Blocks behind a query grid that zero the rows of no sequence (none as a
// rule: they then leave after two loads).
constexpr int kPackedZeroBlocks = 32;

inline int packed_slots(const PackedParams& p, int tile_rows) { return p.T / tile_rows + p.nseq; }

void launch_packed_fwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream);
void launch_packed_bwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream);
void launch_packed_fwd16_wide(const PackedParams& p, int io_dtype, hipStream_t stream);
void launch_packed_bwd16_wide(const PackedParams& p, int io_dtype, hipStream_t stream);
void launch_packed_fwd32(const PackedParams& p, int dp, hipStream_t stream);
void launch_packed_bwd32(const PackedParams& p, int dp, hipStream_t stream);

}  // namespace nxa
