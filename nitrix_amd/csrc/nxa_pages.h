// Parameter blocks and launchers of nxa_pages.hip.
#pragma once

#include "nxa_paged.h"

namespace nxa {

struct WriteParams : PoolParams {
  const void *ks, *vs;         // [Hk, T, D], [Hk, T, Dv]
  int64_t ks_str[2], vs_str[2];  // head, token
  const int* offsets;          // [B + 1], or null: token s is sequence s's
  const int* starts;           // [B]
  const int* table;
  int64_t table_rs;
  int64_t T;
  int B, M, es;
};

// Page pairs in kernel arguments: no copy to the device, no buffer to keep.
constexpr int kCopyPairs = 400;
struct CopyPairs {
  int n;
  int src[kCopyPairs], dst[kCopyPairs];
};

struct StartParams {
  const int* src[3];
  int* dst[3];
  int64_t n[3];
};

// Free, extend and fork: contiguous [B, M] tables.
struct RowsParams {
  const int *table, *lengths, *refs;
  int *table_out, *lengths_out, *refs_out;
  const int* rows;    // free: rows; fork: sources (n of them)
  const int* counts;  // extend: new tokens [B]; fork: targets
  int* work;          // extend: [P]; fork: [n + B + min(n, P)]
  int B, M, P, PS, n;
  int start;          // the kernel itself copies what the results start from
};

// Up to so many numbers a single block copies the state itself: free, fork and
// extend of 64 rows of 128 entries and 4096 pages, 66 -> 57 us a step, most of
// it on the host, with three launches less.
constexpr int64_t kStartAlone = 32768;
constexpr int kFreeAlone = 1024;  // rows that the single block frees
// Columns of a grown row that a thread takes alone, a row's wave 64 a step.  us
// in a graph, thread / wave: 64 rows of 12 columns 15 / 17, 24 20 / 17, 48 33 / 17,
// 500 246 / 51; 512 of 12 24 / 62, 100 172 / 108; one of 6000 1723 / 66.
constexpr int kLaneColumns = 32;

constexpr int kCompactPages = 4096;  // pages of a counting block
constexpr int kCompactFew = 8;
struct CompactParams {
  const int *table, *refs;
  int *table_out, *refs_out;
  int *counts, *info, *movers, *holes, *mover_rank;  // workspace
  int64_t entries;
  int P, Hk, PS;
};

void launch_pages_write(const WriteParams& p, hipStream_t stream);
void launch_pages_copy(const PoolParams& p, int es, const CopyPairs& pairs, hipStream_t stream);
void launch_pages_free(const RowsParams& p, hipStream_t stream);
void launch_pages_extend(RowsParams p, hipStream_t stream);
void launch_pages_fork(RowsParams p, const PoolParams& pool, int es, hipStream_t stream);
void launch_pages_compact(const CompactParams& p, const PoolParams& pool, int es,
                          hipStream_t stream);

}  // namespace nxa
