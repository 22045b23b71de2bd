// How the blocks of a paged attention share the work, and the loads that feed
// it: device code of nxa_paged.hip and nxa_qpaged.hip.
#pragma once

#include "nxa_paged.h"

namespace nxa {

namespace {

// (the running maximum is raised in steps of more than 2^kSlack)
constexpr float kSlack = 8.0f;
constexpr int kWaves = 4;

__device__ __forceinline__ float xor16(float x) { return __shfl_xor(x, 16, 64); }

// Tokens of sequence b, and tiles of so many.
__device__ __forceinline__ int paged_len(const PagedParams& p, int b) {
  // (a length beyond the table's room counts as the room)
  const int64_t room = (int64_t)p.M * p.PS;
  const int n = p.lengths[b];
  return n < 0 ? 0 : n > room ? (int)room : n;
}
__device__ __forceinline__ int paged_tiles(int len) {
  return (int)(((int64_t)len + kPagedKeys - 1) / kPagedKeys);
}
// Units of a (sequence, head): its tiles after START for starting on it.
template <int START>
__device__ __forceinline__ int paged_units(const PagedParams& p, int b) {
  const int n = paged_tiles(paged_len(p, b));
  return n ? n + START : 0;
}
// Sum of the sequences' units a head before each of 256 consecutive groups of
// sequences, into pre[0 .. 256] (LDS).
template <int START>
__device__ __forceinline__ void paged_prefix(const PagedParams& p, int* pre, int* wsum) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (p.B + 255) / 256;
  int n = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < p.B) n += paged_units<START>(p, tid * per + i);
  int x = n;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  if (lane == 63) wsum[wave] = x;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) base += w < wave ? wsum[w] : 0;
  pre[tid + 1] = base + x;
  if (tid == 0) pre[0] = 0;
  __syncthreads();
}

// Blocks that get work: at most one a unit, so that none of them is empty
// (the join takes a piece from every block between a row's first and last).
__device__ __forceinline__ int busy_blocks(const PagedParams& p, int64_t units) {
  return (int)min((int64_t)p.nblk, units);
}
// o of a sequence without tokens.
template <typename T>
__device__ __forceinline__ void paged_zero(const PagedParams& p, int b) {
  T* op = (T*)p.o + b * p.o_str[0];
  for (int i = threadIdx.x; i < p.Hk * p.G * p.Dv; i += 256)
    op[(i / p.Dv) * p.o_str[1] + i % p.Dv] = (T)0.f;
}
// First unit of block i of n.
__device__ __forceinline__ int64_t first_unit(int64_t units, int i, int n) { return units * i / n; }

constexpr int kNonTemporal = 2;  // cache policy of a buffer load

// N dwords from a buffer resource at a byte offset (zero past its end).
template <int N>
struct Words {
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> buf_load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  Words<N> x;
  if constexpr (N == 1) {
    x.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, kNonTemporal);
  } else if constexpr (N == 2) {
    const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, kNonTemporal);
    x.w[0] = y[0], x.w[1] = y[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * i, 0, kNonTemporal);
#pragma unroll
      for (int j = 0; j < 4; ++j) x.w[i + j] = y[j];
    }
  }
  return x;
}

}  // namespace

}  // namespace nxa
