// Paged key-value cache: parameter blocks and launchers of nxa_paged.hip (one
// new token a sequence attends its pages) and nxa_pages.hip (writing, copying
// and managing pages).
//
// A pool holds P pages of PS token slots for each of Hk heads: k [P, Hk, PS,
// D], v [P, Hk, PS, Dv], unit stride over the head dim.  Row b of a page table
// [B, M] lists a sequence's pages in order: its token j is slot j % PS of page
// table[b][j / PS].  An entry outside 0 .. P - 1 is no page: it is never
// followed, so whatever a table holds, no access leaves the pool.
#pragma once

#include "nxa_common.h"

namespace nxa {

struct PoolParams {
  void *k, *v;
  int64_t k_str[3], v_str[3];  // page, head, slot (elements)
  int P, Hk, PS, D, Dv;
};

struct PagedParams : PoolParams {
  const void* q;     // [B, Hk * G, D]
  void* o;           // [B, Hk * G, Dv]
  int64_t q_str[2], o_str[2];  // sequence, head
  const int* table;
  const int* lengths;
  int64_t table_rs;
  int B, M, G;
  int strips;        // of 16 query heads that share a key-value head
  int nblk;          // blocks that share the work; 0: a block a row
  float scale_log2;
  float* part;       // [2 nblk] partial results (paged_part_floats each)
  int4* joins;       // [nblk] the row that starts in a block and goes on in the next:
                     // sequence, head, pieces (0: none), its first piece
};

constexpr int kPagedKeys = 128;    // keys of a work unit
constexpr int kStartUnits = 1;     // what starting on a row costs, in units
constexpr int kPagedBlocks = 512;  // most blocks that share the work
constexpr int kJoinPieces = 768;   // most of any kernel whose pieces are joined
// One partial result: [16 heads][DP] sums, then a maximum and a sum a head.
constexpr int paged_part_floats(int dp) { return 16 * dp + 32; }
int paged_dp(int m);               // padded head dim
// Whether a block takes a whole row (sequence and key-value head) of up to
// `room` tokens; else as many share the units as there are, at most kPagedBlocks.
bool paged_whole(int64_t room);
void launch_paged(const PagedParams& p, int io_dtype, hipStream_t stream);
// The second kernel alone, for pieces of dp = 64, 128 or 256 columns.
void launch_paged_join(const PagedParams& p, int io_dtype, int dp, hipStream_t stream);

}  // namespace nxa
