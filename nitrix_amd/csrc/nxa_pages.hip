// Writing, copying and managing the pages of a key-value cache (nxa_paged.h).
//
// All of it moves rows of whole 16-byte chunks, bound by HBM where there is
// much of it and by launches where there is little.  The tables, lengths and
// reference counts are read on the device and results go to arrays of their
// own, so nothing here waits for the host.  Page ids, row numbers and lengths
// are checked where they are read: one outside its range is skipped.
#include "nxa_pages.h"

namespace nxa {

namespace {

// Rows of `cpr` 16-byte chunks, threads laid over (row, chunk): rows r0, r0 +
// step, ... of a block of `threads` threads.
struct RowWalk {
  int r0, step, c;
  __device__ __forceinline__ RowWalk(int cpr, int tid, int threads) {
    step = threads / cpr;
    r0 = tid / cpr;
    c = tid - r0 * cpr;
    if (r0 >= step) r0 = INT32_MAX;  // left over
  }
};

__device__ __forceinline__ void copy_rows(char* dst, const char* src, int rows, int cpr,
                                          int64_t stride, int tid, int threads) {
  // (one chunk a step and thread; four in flight)
  const RowWalk w(cpr, tid, threads);
  int64_t off = (int64_t)w.r0 * stride + 16 * w.c;
  int r = w.r0;
  const int64_t hop = (int64_t)w.step * stride;
  for (; r < rows - 3 * w.step && r < rows; r += 4 * w.step, off += 4 * hop) {
    u32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const u32x4*>(src + off + i * hop);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(dst + off + i * hop) = x[i];
  }
  for (; r < rows; r += w.step, off += hop)
    *reinterpret_cast<u32x4*>(dst + off) = *reinterpret_cast<const u32x4*>(src + off);
}

// `rows` slots of one head of page `from` to page `to`, keys and values.
__device__ __forceinline__ void copy_head(const PoolParams& p, int es, int from, int to, int head,
                                          int rows, int tid, int threads) {
  char* k = (char*)p.k + head * p.k_str[1] * es;
  char* v = (char*)p.v + head * p.v_str[1] * es;
  copy_rows(k + to * p.k_str[0] * es, k + from * p.k_str[0] * es, rows, p.D * es / 16,
            p.k_str[2] * es, tid, threads);
  copy_rows(v + to * p.v_str[0] * es, v + from * p.v_str[0] * es, rows, p.Dv * es / 16,
            p.v_str[2] * es, tid, threads);
}

__device__ __forceinline__ bool is_page(int e, int P) { return (unsigned)e < (unsigned)P; }

// Inclusive sum over a block of 1024 threads; `total` the block's.
__device__ __forceinline__ int block_scan(int x, int* wsum, int& total) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nw = blockDim.x / 64;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) wsum[wave] = x;
  __syncthreads();
  int base = 0;
  total = 0;
  for (int w = 0; w < nw; ++w) {
    base += w < wave ? wsum[w] : 0;
    total += wsum[w];
  }
  return base + x;
}

// The first `need` free pages (refs <= 0), lowest first, into list; returns
// how many there are of them.  One block of 1024 threads.
__device__ int find_free(const int* refs, int P, int need, int* list, int* wsum) {
  int found = 0;
  for (int p0 = 0; p0 < P && found < need; p0 += 4096) {
    const int at = p0 + 4 * threadIdx.x;
    int fr[4], n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fr[i] = at + i < P && refs[at + i] <= 0;
      n += fr[i];
    }
    int total;
    int rank = found + block_scan(n, wsum, total) - n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (fr[i]) {
        if (rank < need) list[rank] = at + i;
        ++rank;
      }
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

// The state that the results start from, by one block of 1024 threads, whose
// later writes and counts come after it.
__device__ __forceinline__ void start_alone(const RowsParams& p) {
  auto copy = [](int* dst, const int* src, int n) NXA_INLINE {
    int done = 0;
    if ((((uintptr_t)dst | (uintptr_t)src) & 15) == 0) {
      done = n & ~3;
#pragma unroll 4
      for (int i = 4 * threadIdx.x; i < done; i += 4096)
        *reinterpret_cast<int4*>(dst + i) = *reinterpret_cast<const int4*>(src + i);
    }
    for (int i = done + threadIdx.x; i < n; i += 1024) dst[i] = src[i];
  };
  copy(p.table_out, p.table, p.B * p.M);
  copy(p.refs_out, p.refs, p.P);
  copy(p.lengths_out, p.lengths, p.B);
  __threadfence();
  __syncthreads();
}

}  // namespace

// ---------------------------------------------------------------------------
// New tokens into their pages, a wave each: it finds the token's sequence (64
// probes a step among the offsets) and page, and moves the rows of every head.
// Bound by HBM: 16384 tokens of 8 heads of 128, 67 MB read and written, 27 us
// (5.0 TB/s, the rate of a copy).  2 and 4 tokens a wave, one after the other,
// wait for one another's lookups (34 and 36 us, 30.5 with one); the rows are
// read once, past the caches (30.5 -> 27).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void pages_write_kernel(const WriteParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.T) return;
  const int ck = p.D * p.es / 16, cv = p.Dv * p.es / 16, all = p.Hk * (ck + cv);
  int s = (int)t;
  int64_t pos = 0;
  if (p.offsets) {
    int lo = 0, hi = p.B + 1;  // last s with offsets[s] <= t
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64;
      const int x = lo + lane * step;
      const int cnt = (int)__popcll(__ballot(x < hi && p.offsets[x] <= t));
      if (cnt == 0) break;  // before the first sequence
      lo += (cnt - 1) * step;
      hi = min(lo + step, hi);
    }
    s = __builtin_amdgcn_readfirstlane(lo);
    if (s >= p.B || p.offsets[s] > t) return;
    pos = t - p.offsets[s];
  }
  pos += p.starts[s];
  if (pos < 0 || pos >= (int64_t)p.M * p.PS) return;
  const int page = p.table[s * p.table_rs + pos / p.PS];
  if (!is_page(page, p.P)) return;
  const int slot = (int)(pos % p.PS);
  const char* ks = (const char*)p.ks + t * p.ks_str[1] * p.es;
  const char* vs = (const char*)p.vs + t * p.vs_str[1] * p.es;
  char* kd = (char*)p.k + (page * p.k_str[0] + slot * p.k_str[2]) * p.es;
  char* vd = (char*)p.v + (page * p.v_str[0] + slot * p.v_str[2]) * p.es;
#pragma unroll 4
  for (int x = lane; x < all; x += 64) {
    const bool key = x < p.Hk * ck;
    const int y = key ? x : x - p.Hk * ck, cpr = key ? ck : cv;
    const int h = y / cpr, c = 16 * (y - h * cpr);
    const char* src = key ? ks + h * p.ks_str[0] * p.es : vs + h * p.vs_str[0] * p.es;
    char* dst = key ? kd + h * p.k_str[1] * p.es : vd + h * p.v_str[1] * p.es;
    *reinterpret_cast<u32x4*>(dst + c) =
        __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + c));
  }
}

// ---------------------------------------------------------------------------
// Page copies named by the host, a block a (pair, head).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void pages_copy_kernel(const PoolParams p, int es,
                                                         const CopyPairs pairs) {
  const int i = blockIdx.x / p.Hk, h = blockIdx.x % p.Hk;
  copy_head(p, es, pairs.src[i], pairs.dst[i], h, p.PS, threadIdx.x, 256);
}

// Copies of up to three int arrays (the tables an operation starts from).
__global__ __launch_bounds__(256) void pages_start_kernel(const StartParams p) {
  for (int a = 0; a < 3; ++a) {
    const int64_t n = p.n[a];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
      p.dst[a][i] = p.src[a][i];
  }
}

// ---------------------------------------------------------------------------
// Rows given back: a block a listed row (the first time it is listed).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void pages_free_kernel(const RowsParams p) {
  __shared__ int again;
  const int tid = threadIdx.x, r = p.rows[blockIdx.x];
  if ((unsigned)r >= (unsigned)p.B) return;
  if (tid == 0) again = 0;
  __syncthreads();
  for (int i = tid; i < (int)blockIdx.x; i += 256)
    if (p.rows[i] == r) again = 1;
  __syncthreads();
  if (again) return;
  for (int c = tid; c < p.M; c += 256) {
    const int e = p.table[(int64_t)r * p.M + c];
    if (is_page(e, p.P)) atomicAdd(p.refs_out + e, -1);
    p.table_out[(int64_t)r * p.M + c] = -1;
  }
  if (tid == 0) p.lengths_out[r] = 0;
}

// The same by one block, of up to kFreeAlone rows.
__global__ __launch_bounds__(1024) void pages_free_alone_kernel(const RowsParams p) {
  __shared__ int rows[kFreeAlone];
  const int tid = threadIdx.x, lane = tid & 63;
  const int mine = tid < p.n ? p.rows[tid] : -1;
  rows[tid] = mine;
  start_alone(p);
  bool first = (unsigned)mine < (unsigned)p.B;
  for (int i = 0; i < tid && first; ++i) first = rows[i] != mine;
  __syncthreads();
  rows[tid] = first ? mine : -1;
  __syncthreads();
  for (int i = tid >> 6; i < p.n; i += 16) {
    const int r = rows[i];
    if (r < 0) continue;
    for (int c = lane; c < p.M; c += 64) {
      const int e = p.table[(int64_t)r * p.M + c];
      if (is_page(e, p.P)) atomicAdd(p.refs_out + e, -1);
      p.table_out[(int64_t)r * p.M + c] = -1;
    }
    if (lane == 0) p.lengths_out[r] = 0;
  }
}

// ---------------------------------------------------------------------------
// Rows grown: the new tokens' missing pages are numbered through in row and
// column order and the k-th takes the k-th free page.  One block: a thread
// takes its rows' columns one after the other (a new token or a few reach one
// or two); rows whose tokens reach more than kLaneColumns (prompts) are taken
// by a wave each, 64 columns a step, their counts and first ranks passed
// through lengths_out.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void pages_extend_kernel(const RowsParams p) {
  __shared__ int wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (p.start) start_alone(p);
  const int per = (p.B + 1023) / 1024;
  const int64_t room = (int64_t)p.M * p.PS;
  // Columns [first, last) of row r that its new tokens reach.
  auto span = [&](int r, int& first, int& last, int64_t& grown) {
    const int64_t len = min(max((int64_t)p.lengths[r], (int64_t)0), room);
    grown = min(len + max(p.counts[r], 0), room);
    first = (int)((len + p.PS - 1) / p.PS);
    last = (int)((grown + p.PS - 1) / p.PS);
  };
  auto missing = [&](int r, int64_t c) { return !is_page(p.table[(int64_t)r * p.M + c], p.P); };
  int need = 0;
  bool wide = false;
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r >= p.B) break;
    int a, b;
    int64_t g;
    span(r, a, b, g);
    if (b - a > kLaneColumns) {
      wide = true;
      continue;
    }
    for (int c = a; c < b; ++c) need += missing(r, c);
  }
  wide = __syncthreads_or(wide);
  if (wide) {
    for (int r = wave; r < p.B; r += 16) {
      int a, b, n = 0;
      int64_t g;
      span(r, a, b, g);
      if (b - a <= kLaneColumns) continue;
#pragma unroll 4
      for (int64_t c = a; c < b; c += 64)
        n += (int)__popcll(__ballot(c + lane < b && missing(r, min(c + lane, (int64_t)b - 1))));
      if (lane == 0) p.lengths_out[r] = n;
    }
    __syncthreads();
    for (int i = 0; i < per; ++i) {
      const int r = tid * per + i;
      if (r >= p.B) break;
      int a, b;
      int64_t g;
      span(r, a, b, g);
      if (b - a > kLaneColumns) need += p.lengths_out[r];
    }
  }
  int total;
  int rank = block_scan(need, wsum, total) - need;
  const int got = find_free(p.refs, p.P, min(total, p.P), p.work, wsum);
  __threadfence_block();
  // Column c of row r without a page, the k-th of all; false where the pages
  // have run out.
  auto take = [&](int r, int64_t c, int k) {
    const int page = k < got ? p.work[k] : -1;
    p.table_out[(int64_t)r * p.M + c] = page;
    if (page >= 0) p.refs_out[page] = 1;
    return page >= 0;
  };
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r >= p.B) break;
    int a, b;
    int64_t g;
    span(r, a, b, g);
    if (b - a > kLaneColumns) {
      const int n = p.lengths_out[r];
      p.lengths_out[r] = rank;
      rank += n;
      continue;
    }
    for (int c = a; c < b; ++c) {
      if (!missing(r, c)) continue;
      // Out of pages: the row ends with the tokens that have one.
      if (!take(r, c, rank)) g = min(g, (int64_t)c * p.PS);
      ++rank;
    }
    p.lengths_out[r] = (int)g;
  }
  if (!wide) return;
  __syncthreads();
  for (int r = wave; r < p.B; r += 16) {
    int a, b;
    int64_t g;
    span(r, a, b, g);
    if (b - a <= kLaneColumns) continue;
    int k = p.lengths_out[r];
    for (int64_t c0 = a; c0 < b; c0 += 64) {
      const int64_t c = c0 + lane;
      const bool miss = c < b && missing(r, c);
      const uint64_t m = __ballot(miss);
      bool out = false;
      if (miss) out = !take(r, c, k + (int)__popcll(m & ((1ull << lane) - 1)));
      const uint64_t none = __ballot(out);
      if (none) g = min(g, (c0 + (int)__builtin_ctzll(none)) * p.PS);
      k += (int)__popcll(m);
    }
    if (lane == 0) p.lengths_out[r] = (int)g;
  }
}

// ---------------------------------------------------------------------------
// Forks.  First a block settles which entries count (of those that name one
// row as their target the last) and gives each that needs it a free page.
// work[i]: -2 does not count, -1 no page needed (or none left), else the page.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void pages_fork_plan_kernel(const RowsParams p) {
  __shared__ int wsum[16];
  const int tid = threadIdx.x;
  if (p.start) start_alone(p);
  int* winner = p.work + p.n;          // [B]
  int* list = winner + p.B;            // [min(n, P)]
  for (int r = tid; r < p.B; r += 1024) winner[r] = -1;
  __syncthreads();
  auto counts = [&](int i) {
    const int s = p.rows[i], d = p.counts[i];
    return (unsigned)s < (unsigned)p.B && (unsigned)d < (unsigned)p.B && s != d;
  };
  for (int i = tid; i < p.n; i += 1024)
    if (counts(i)) atomicMax(winner + p.counts[i], i);
  __syncthreads();
  const int per = (p.n + 1023) / 1024;
  const int64_t room = (int64_t)p.M * p.PS;
  // (a partly filled last page of a source that has that page)
  auto wants = [&](int i) {
    const int s = p.rows[i];
    const int64_t len = min(max((int64_t)p.lengths[s], (int64_t)0), room);
    return len % p.PS != 0 && is_page(p.table[(int64_t)s * p.M + len / p.PS], p.P);
  };
  int need = 0;
  for (int k = 0; k < per; ++k) {
    const int i = tid * per + k;
    if (i >= p.n) break;
    if (counts(i) && winner[p.counts[i]] == i) need += wants(i);
  }
  int total;
  int rank = block_scan(need, wsum, total) - need;
  const int got = find_free(p.refs, p.P, min(total, p.P), list, wsum);
  for (int k = 0; k < per; ++k) {
    const int i = tid * per + k;
    if (i >= p.n) break;
    int w = -2;
    if (counts(i) && winner[p.counts[i]] == i) {
      w = -1;
      if (wants(i)) {
        if (rank < got) w = list[rank];
        ++rank;
      }
    }
    p.work[i] = w;
  }
}

// Then blocks (i, 0) write the rows and counts, and blocks (i, 1 + h) copy
// head h of the partly filled last page.
__global__ __launch_bounds__(256) void pages_fork_kernel(const RowsParams p, const PoolParams pool,
                                                         int es) {
  const int i = blockIdx.x, tid = threadIdx.x;
  const int fresh = p.work[i];
  if (fresh == -2) return;
  const int s = p.rows[i], d = p.counts[i];
  const int64_t room = (int64_t)p.M * p.PS;
  const int len = (int)min(max((int64_t)p.lengths[s], (int64_t)0), room);
  const int full = len / p.PS, rest = len % p.PS;
  if (blockIdx.y > 0) {
    if (fresh < 0) return;
    const int from = p.table[(int64_t)s * p.M + full];
    if (is_page(from, p.P)) copy_head(pool, es, from, fresh, blockIdx.y - 1, rest, tid, 256);
    return;
  }
  for (int c = tid; c < p.M; c += 256) {
    const int old = p.table[(int64_t)d * p.M + c];
    if (is_page(old, p.P)) atomicAdd(p.refs_out + old, -1);
    int e = -1;
    if (c < full) e = p.table[(int64_t)s * p.M + c];
    else if (c == full) e = fresh;
    if (is_page(e, p.P)) atomicAdd(p.refs_out + e, 1);
    else e = -1;
    p.table_out[(int64_t)d * p.M + c] = e;
  }
  if (tid == 0) p.lengths_out[d] = rest && fresh < 0 ? full * p.PS : len;
}

// ---------------------------------------------------------------------------
// Compaction.  n live pages: the k-th live page from n on moves into the k-th
// dead one below n.  Blocks of kCompactPages pages are counted; then each block
// adds up the counts before it and lists its movers and holes; then pages,
// table and counts move.  (Up to kCompactFew blocks count for themselves: a
// launch of 3 us less.)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void pages_count_kernel(const CompactParams p) {
  __shared__ int wsum[16];
  const int at = blockIdx.x * kCompactPages + 4 * threadIdx.x;
  int n = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) n += at + i < p.P && p.refs[at + i] > 0;
  int total;
  block_scan(n, wsum, total);
  if (threadIdx.x == 0) p.counts[blockIdx.x] = total;
}

__global__ __launch_bounds__(1024) void pages_plan_kernel(const CompactParams p) {
  __shared__ int wsum[16];
  const int tid = threadIdx.x, nb = (p.P + kCompactPages - 1) / kCompactPages;
  const bool few = nb <= kCompactFew;  // (then not counted before)
  // Live pages in all (n) and before this block.
  int part[2] = {0, 0};
  if (few) {
    for (int i = 0; i < nb; ++i) {
      int c = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = i * kCompactPages + 4 * tid + e;
        c += at < p.P && p.refs[at] > 0;
      }
      part[0] += c;
      part[1] += i < (int)blockIdx.x ? c : 0;
    }
  } else {
    for (int i = tid; i < nb; i += 1024) {
      part[0] += p.counts[i];
      part[1] += i < (int)blockIdx.x ? p.counts[i] : 0;
    }
  }
  int n, before;
  block_scan(part[0], wsum, n);
  block_scan(part[1], wsum, before);
  // Live pages below n: those before its block and those of its block.
  const int bn = n / kCompactPages;
  int x = 0;
  if (few) {
    for (int i = 0; i < bn; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x += p.refs[i * kCompactPages + 4 * tid + e] > 0;
  } else {
    for (int i = tid; i < bn; i += 1024) x += p.counts[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = bn * kCompactPages + 4 * tid + i;
    x += at < n && p.refs[at] > 0;
  }
  int low;
  block_scan(x, wsum, low);
  int live[4], m = 0;
  const int at = blockIdx.x * kCompactPages + 4 * tid;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    live[i] = at + i < p.P && p.refs[at + i] > 0;
    m += live[i];
  }
  int total;
  int rank = before + block_scan(m, wsum, total) - m;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int page = at + i;
    if (page < p.P) {
      if (page >= n && live[i]) {
        p.movers[rank - low] = page;
        p.mover_rank[page] = rank - low;
      }
      if (page < n && !live[i]) p.holes[page - rank] = page;
    }
    rank += live[i];
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.info[0] = n;
    p.info[1] = n - low;  // movers
  }
}

__global__ __launch_bounds__(256) void pages_move_kernel(const CompactParams p,
                                                         const PoolParams pool, int es) {
  const int tid = threadIdx.x;
  const int n = p.info[0], moves = p.info[1];
  auto where = [&](int e) { return e >= n && p.refs[e] > 0 ? p.holes[p.mover_rank[e]] : e; };
  const int64_t stride = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + tid;
  for (int64_t i = i0; i < p.entries; i += stride) {
    const int e = p.table[i];
    p.table_out[i] = is_page(e, p.P) ? where(e) : e;
  }
  for (int64_t i = i0; i < p.P; i += stride) {
    const int r = max(p.refs[i], 0);
    // (a hole's count is written where its mover's is read)
    if (i >= n) {
      p.refs_out[i] = 0;
      if (r > 0) p.refs_out[p.holes[p.mover_rank[i]]] = r;
    } else if (r > 0) {
      p.refs_out[i] = r;
    }
  }
  const int64_t jobs = (int64_t)moves * p.Hk;
  for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x)
    copy_head(pool, es, p.movers[j / p.Hk], p.holes[j / p.Hk], (int)(j % p.Hk), p.PS, tid, 256);
}

// ---------------------------------------------------------------------------
// Launchers.
// ---------------------------------------------------------------------------
void launch_pages_write(const WriteParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(pages_write_kernel, dim3((unsigned)((p.T + 3) / 4)), dim3(256), 0, stream, p);
}

void launch_pages_copy(const PoolParams& p, int es, const CopyPairs& pairs, hipStream_t stream) {
  hipLaunchKernelGGL(pages_copy_kernel, dim3(pairs.n * p.Hk), dim3(256), 0, stream, p, es, pairs);
}

// Whether the one-block kernel of the call copies the state itself; else a
// launch of its own does.
static int launch_start(const RowsParams& p, bool one_block, hipStream_t stream) {
  if (one_block && (int64_t)p.B * p.M + p.P + p.B <= kStartAlone) return 1;
  StartParams s = {};
  s.src[0] = p.table, s.dst[0] = p.table_out, s.n[0] = (int64_t)p.B * p.M;
  s.src[1] = p.refs, s.dst[1] = p.refs_out, s.n[1] = p.P;
  s.src[2] = p.lengths, s.dst[2] = p.lengths_out, s.n[2] = p.B;
  const int64_t most = s.n[0] > s.n[1] ? s.n[0] : s.n[1];
  const int64_t blocks = (most + 1023) / 1024;
  hipLaunchKernelGGL(pages_start_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256),
                     0, stream, s);
  return 0;
}

void launch_pages_free(const RowsParams& p, hipStream_t stream) {
  if (launch_start(p, p.n <= kFreeAlone, stream))
    hipLaunchKernelGGL(pages_free_alone_kernel, dim3(1), dim3(1024), 0, stream, p);
  else if (p.n > 0) hipLaunchKernelGGL(pages_free_kernel, dim3(p.n), dim3(256), 0, stream, p);
}

void launch_pages_extend(RowsParams p, hipStream_t stream) {
  p.start = launch_start(p, true, stream);
  hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(1024), 0, stream, p);
}

void launch_pages_fork(RowsParams p, const PoolParams& pool, int es, hipStream_t stream) {
  p.start = launch_start(p, p.n > 0, stream);
  if (p.n == 0) return;
  hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(1), dim3(1024), 0, stream, p);
  hipLaunchKernelGGL(pages_fork_kernel, dim3(p.n, 1 + pool.Hk), dim3(256), 0, stream, p, pool, es);
}

void launch_pages_compact(const CompactParams& p, const PoolParams& pool, int es,
                          hipStream_t stream) {
  const int nb = (p.P + kCompactPages - 1) / kCompactPages;
  if (nb > kCompactFew)
    hipLaunchKernelGGL(pages_count_kernel, dim3(nb), dim3(1024), 0, stream, p);
  hipLaunchKernelGGL(pages_plan_kernel, dim3(nb), dim3(1024), 0, stream, p);
  hipLaunchKernelGGL(pages_move_kernel, dim3(2048), dim3(256), 0, stream, p, pool, es);
}

}  // namespace nxa
