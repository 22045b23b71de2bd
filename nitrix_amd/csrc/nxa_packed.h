// Packed sequences: several sequences laid end to end along the token axis,
// sequence s at rows offsets[s] .. offsets[s + 1] - 1, and G query heads to
// each key-value head.  The attention kernels take a PackedParams in place
// of Params; each block finds its (sequence, tile, head) here and then works
// on that sequence as on a dense problem of one head.
//
// A grid needs an upper bound of the tiles without the lengths, which are on
// the device: floor(T / TILE) + (sequences) tiles of TILE rows are always
// enough.
//
// Up to kRankedSeqs sequences are taken in order of work, the longest tiles
// of all sequences and heads first, so that none of them starts late: block i
// takes the i-th tile by descending index (causal; the number of tiles from
// index j on, f(j) = sum_s max(0, tiles_s - j), is a sum over lanes, and j a
// binary search) or by descending length of its sequence.  With more of them a
// wave finds the sequence of slot i without any sum: sequence s owns the
// slots from S(s) = floor(offsets[s] / TILE) + s on, which grow by at least
// ceil(length / TILE) from one sequence to the next, and S is monotone, so
// ballots over 64 probes a step find it.
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
  void* o_lo;          // what rounding o to 16 bits left (o's strides), or null
  // dK / dV of a group of query heads in `parts` blocks, each over one or more
  // of them, whose fp32 sums go to dkv_part ([parts][Hk][T][D], then the same of
  // dV) and are added up afterwards (1: one block takes them all).
  int parts;
  float* dkv_part;
};

// What a dK / dV block streams besides its own sequence's base pointers.
struct PackedGroup {
  int heads;                   // query heads of the group (1 or more)
  int64_t q_hs, do_hs, row_hs; // from one head to the next (row_hs: nlse2, ndelta)
  int64_t do_rs, dk_rs, dv_rs; // row strides
  float *dk_part, *dv_part;    // this block's rows of dkv_part, or null
};

struct PackedTile {
  int start, len, tile;
};

__device__ __forceinline__ int packed_offset(const PackedParams& pp, int s) {
  return min(max(pp.offsets[s], 0), pp.T);
}

constexpr int kRankedSeqs = 256;

// Sum over the wave (uniform), by row shifts and broadcasts.
__device__ __forceinline__ int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return __builtin_amdgcn_readlane(x, 63);
}

// The rank-th tile in order of work (all lanes active; uniform results).  A
// rank past the last tile gives length zero.  `keys`: tiles of keys, whose
// causal work falls with the index.
template <bool CAUSAL>
__device__ __forceinline__ PackedTile packed_ranked(const PackedParams& pp, int rank,
                                                    int tile_rows, bool keys) {
  constexpr int N = kRankedSeqs / 64;
  const int lane = threadIdx.x & 63;
  int nt[N], most = 0, total = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int s = lane + 64 * k;
    nt[k] = 0;
    if (s < pp.nseq) {
      const int len = packed_offset(pp, s + 1) - packed_offset(pp, s);
      nt[k] = len > 0 ? (len + tile_rows - 1) / tile_rows : 0;
    }
    most = max(most, nt[k]);
    total += nt[k];
  }
  PackedTile r = {0, 0, 0};
  if (rank >= wave_sum(total)) return r;
  // Tiles with index j or more (causal), or in sequences of more than j tiles.
  auto tiles_from = [&](int j) -> int {
    int x = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) x += CAUSAL ? max(nt[k] - j, 0) : nt[k] > j ? nt[k] : 0;
    return wave_sum(x);
  };
  int lo = 0, hi = 1;
  while (__any(most >= hi)) hi *= 2;  // tiles_from(hi) == 0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tiles_from(mid) > rank) lo = mid;
    else hi = mid;
  }
  // Causal: tiles of index lo; else the sequences of lo + 1 tiles, each with
  // all of its tiles.
  int at = rank - tiles_from(lo + 1), tile = lo;
  if (!CAUSAL) {
    tile = at % (lo + 1);
    at /= lo + 1;
  }
  int seq = 0, cnt = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint64_t m = __ballot(CAUSAL ? nt[k] > lo : nt[k] == lo + 1);
    const int c = __popcll(m);
    if (at >= 0 && at < c) {
      // The at-th set bit.
      const int mine = (int)__popcll(m & ((1ull << lane) - 1));
      const uint64_t hit = __ballot((m >> lane & 1) && mine == at);
      const int l = (int)__builtin_ctzll(hit);
      seq = 64 * k + l;
      cnt = __builtin_amdgcn_readlane(nt[k], l);
    }
    at -= c;
  }
  r.start = __builtin_amdgcn_readfirstlane(packed_offset(pp, seq));
  r.len = __builtin_amdgcn_readfirstlane(packed_offset(pp, seq + 1)) - r.start;
  r.tile = CAUSAL && keys ? cnt - 1 - tile : tile;
  return r;
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
  // (offsets that decrease can end the search at a sequence behind the slot,
  // whose tiles before its first row are other sequences' rows)
  if (r.tile < 0) r.len = r.tile = 0;
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

// Rank and virtual head of block bid: tiles in order, the heads of a tile next
// to each other.  Blocks that run on one XCD (every eighth) share heads, those
// of one key-value head where their number allows, so its tiles meet in L2.
struct PackedBlock {
  int rank, hv;
};
__device__ __forceinline__ PackedBlock packed_block(int bid, int heads) {
  if (heads % 8) return {bid / heads, bid % heads};
  const int x = bid % 8, k = bid / 8, per = heads / 8;
  return {k / per, x + 8 * (k % per)};
}

template <bool CAUSAL>
__device__ __forceinline__ PackedTile packed_tile(const PackedParams& pp, int rank, int rows,
                                                  bool keys) {
  if (pp.nseq <= kRankedSeqs) return packed_ranked<CAUSAL>(pp, rank, rows, keys);
  // (a causal query tile late in its sequence has the most keys, a key tile
  // early in it the most queries)
  return packed_find(pp, keys ? rank : pp.slots - 1 - rank, rows);
}

// The rows of o_lo that go with p.o (a packed problem has no qk-norm, whose
// output pointer carries them).
template <typename T>
__device__ __forceinline__ T* packed_o_lo(const Params& p) {
  return (T*)p.qn_out;
}

// Blocks of the forward and dQ kernels: one query tile of one query head.
// False: nothing to do.
template <typename T, bool CAUSAL>
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
  const PackedBlock blk = packed_block(bid, pp.Hk * pp.G);
  const int hk = blk.hv % pp.Hk, hq = hk * pp.G + blk.hv / pp.Hk;
  const PackedTile t = packed_tile<CAUSAL>(pp, blk.rank, rows, false);
  if ((int64_t)t.tile * rows >= t.len) return false;
  packed_base(pp, p);
  const int64_t r0 = t.start;
  p.q = (const T*)pp.q + hq * pp.q_str[1] + r0 * pp.q_str[2];
  p.k = (const T*)pp.k + hk * pp.k_str[1] + r0 * pp.k_str[2];
  p.v = (const T*)pp.v + hk * pp.v_str[1] + r0 * pp.v_str[2];
  const int64_t ro = hq * pp.o_str[1] + r0 * pp.o_str[2];
  p.o = (T*)pp.o + ro;
  p.qn_out = pp.o_lo ? (T*)pp.o_lo + ro : nullptr;  // (packed_o_lo)
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

// Blocks of the dK / dV kernels: one key tile of one key-value head, for one
// part of the query heads that share it.
template <typename T, bool CAUSAL>
__device__ __forceinline__ bool packed_key_block(const PackedParams& pp, int rows, Params& p,
                                                 int& kt, PackedGroup& grp) {
  const PackedBlock blk = packed_block(blockIdx.x, pp.Hk * pp.parts);
  const int hk = blk.hv % pp.Hk, part = blk.hv / pp.Hk;
  const int per = (pp.G + pp.parts - 1) / pp.parts, h0 = part * per;
  const PackedTile t = packed_tile<CAUSAL>(pp, blk.rank, rows, true);
  if ((int64_t)t.tile * rows >= t.len) return false;
  packed_base(pp, p);
  const int64_t r0 = t.start, hq = (int64_t)hk * pp.G + h0;
  p.q = (const T*)pp.q + hq * pp.q_str[1] + r0 * pp.q_str[2];
  p.k = (const T*)pp.k + hk * pp.k_str[1] + r0 * pp.k_str[2];
  p.v = (const T*)pp.v + hk * pp.v_str[1] + r0 * pp.v_str[2];
  p.dout = (const T*)pp.dout + hq * pp.do_str[1] + r0 * pp.do_str[2];
  p.dk = (T*)pp.dk + hk * pp.dk_str[1] + r0 * pp.dk_str[2];
  p.dv = (T*)pp.dv + hk * pp.dv_str[1] + r0 * pp.dv_str[2];
  p.ndelta = pp.ndelta + hq * pp.T + r0;
  p.nlse2 = pp.nlse2 + hq * pp.T + r0;
  p.Lq = p.Lk = t.len;
  grp.heads = min(per, pp.G - h0);
  grp.dk_part = grp.dv_part = nullptr;
  if (pp.parts > 1) {
    const int64_t row = ((int64_t)part * pp.Hk + hk) * pp.T + r0;
    grp.dk_part = pp.dkv_part + row * pp.D;
    grp.dv_part = pp.dkv_part + (int64_t)pp.parts * pp.Hk * pp.T * pp.D + row * pp.Dv;
    if constexpr (sizeof(T) == 4) p.dk = grp.dk_part, p.dv = grp.dv_part;
  }
  grp.q_hs = pp.q_str[1], grp.do_hs = pp.do_str[1], grp.row_hs = pp.T;
  grp.do_rs = pp.do_str[2];
  grp.dk_rs = pp.parts > 1 ? pp.D : pp.dk_str[2];
  grp.dv_rs = pp.parts > 1 ? pp.Dv : pp.dv_str[2];
  kt = t.tile;
  return true;
}

// Blocks behind a query grid that zero the rows of no sequence (none as a
// rule: they then leave after two loads).
constexpr int kPackedZeroBlocks = 32;

// Parts of dK / dV.  N equal sequences have Hk G T^2 / (2 * 128 * 64 N) steps
// in all and G T / (64 N) in the longest block, so that the mean of 256 CUs is
// Hk T / 65536 longest blocks: parts bring it to one, or to two where long
// sequences of different lengths let single blocks run on alone; each part
// costs another copy of dK and dV in fp32, written and read.  Causal bf16, head
// dim 128, us of the backward with 1, 2, 4 (, 8) parts: 4 key-value heads of 4,
// 16384 tokens, one sequence 3425, 3428, 3467, ragged ones of 1 to 6348 1010,
// 887, 943, of 2048 504, 546, 620, of 512 218, 289, 362; 2 of 8, one sequence
// of 4096 770, 464, 329, 283; 1 of 8, 16384 tokens, ragged 1198, 733, 522, 477,
// of 512 164, 140, 140, 179.
inline int packed_parts(const PackedParams& p) {
  const int64_t mean = (int64_t)p.Hk * p.T;
  const int64_t want = p.T / p.nseq >= 1024 ? 131072 : 65536;
  const int64_t parts = (want + mean - 1) / mean;
  // (as many as it takes with the heads of the largest: none without a head)
  const int per = parts < p.G ? (int)((p.G + parts - 1) / parts) : 1;
  return (p.G + per - 1) / per;
}
inline size_t packed_part_floats(const PackedParams& p) {
  const int parts = packed_parts(p);
  return parts > 1 ? (size_t)parts * p.Hk * p.T * (p.D + p.Dv) : 0;
}
void launch_packed_parts(const PackedParams& p, int io_dtype, hipStream_t stream);

inline int packed_slots(const PackedParams& p, int tile_rows) { return p.T / tile_rows + p.nseq; }
// Threads of a launch with a block a slot of `heads` heads (and the zeroing
// ones), and of the largest launch of a forward and of a backward: a grid holds
// less than 2^32.
inline int64_t packed_threads(const PackedParams& p, int64_t heads, int tile_rows, int threads) {
  return (heads * ((int64_t)p.T / tile_rows + p.nseq) + kPackedZeroBlocks) * threads;
}
int64_t packed_fwd_threads(const PackedParams& p, int io_dtype, int dp);
int64_t packed_bwd_threads(const PackedParams& p, int io_dtype, int dp);
int64_t packed_fwd32_threads(const PackedParams& p, int dp);
int64_t packed_bwd32_threads(const PackedParams& p, int dp);

void launch_packed_fwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream);
void launch_packed_bwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream);
void launch_packed_fwd16_wide(const PackedParams& p, int io_dtype, hipStream_t stream);
void launch_packed_bwd16_wide(const PackedParams& p, int io_dtype, hipStream_t stream);
void launch_packed_fwd32(const PackedParams& p, int dp, hipStream_t stream);
void launch_packed_bwd32(const PackedParams& p, int dp, hipStream_t stream);

}  // namespace nxa
