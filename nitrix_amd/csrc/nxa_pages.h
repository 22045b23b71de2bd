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

// Up to so many numbers a single block copies the state itself, which saves a
// launch and the host 2 to 3 us of it.  us a call of free, fork, extend, alone /
// with the launch: 4112 numbers 15.0 / 17.2, 26.0 / 28.6, 16.3 / 18.8; 28448 14.4 /
// 16.7, 25.4 / 28.1, 16.0 / 18.6; 36928 14.3 / 16.7, 25.5 / 28.1, 16.0 / 18.5; 65600
// 18.4 / 16.7, 25.5 / 28.1, 16.1 / 18.7; 196736 37.4 / 17.1, 27.7 / 28.0, 20.7 / 18.7.
// (In a captured graph, without the host, the launch is the faster: 7.3 / 4.9,
// 12.1 / 10.5, 7.7 / 6.1 at 4112, 11.2 / 4.8, 14.4 / 11.1, 9.5 / 6.1 at 28448.)
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
