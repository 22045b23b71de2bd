// Attention of one new token a sequence over a paged key-value cache.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the sequence's tokens, per query
// head; G query heads read one key-value head.  Every key and value is read
// once and meets 4 G operations a byte (16 bits), so HBM bounds the call and
// the kernel is built to keep loads in flight:
//
//  * Work is split by what there is of it.  A unit is 128 tokens of one
//    (sequence, key-value head); the units of all sequences, which only the
//    device knows, are numbered through and shared evenly by at most 512
//    blocks (two a CU): block i takes units [U i / N, U (i + 1) / N), whatever
//    sequences these belong to.  One long sequence and many ragged ones load
//    the chip alike.  Starting on a row counts as one unit more (64 sequences of
//    up to 8192 tokens 112 -> 102 us, 256 of up to 2048 166 -> 139).  A
//    (sequence, head) that one block holds whole is finished there; the pieces
//    of the others (at most two a block) go to the workspace, and a second
//    kernel joins them in order.  Where the table has room for few tokens
//    (paged_whole) each row is a block's own and nothing is joined.
//  * K and V go from memory to registers in the layout that the matrix
//    instructions read: no LDS, no barrier in the loop, and each of a
//    block's four waves streams its own tokens with NB steps of 16 tokens
//    in flight, past the caches (each row is read once): 64 sequences of up to
//    8192 tokens, 578 MB, 131 -> 122 us, 150,000 tokens of two, 613 MB, 120 ->
//    107 us (5.7 TB/s); 4 steps in flight against 3: 122 -> 119 us, 5: 148.
//  * S^T = K Q^T (16x16 products): a lane's A operand is 16 bytes of one key's
//    row, loaded as they are.  O^T = V^T P^T needs four keys of one column in a
//    lane: lane (g, c) loads DPL = DP / 16 columns from DPL c on of keys 4 g ..
//    4 g + 3 and interleaves them (v_perm); S^T's accumulator holds P^T for
//    just these keys, so P never leaves its lane.
//  * Loads go through buffer resources that end at the step's last token (and
//    are empty where the table has no page): what lies behind a sequence, be it
//    NaN, reads as zero.
//
// The running maximum of a head is raised only when a score exceeds it by
// more than 2^kSlack; sums and outputs accumulate against the same maximum in
// fp32.  In 16 bits P enters the second product as a pair of terms, so that of
// its rounding 2^-16 (bf16) is left; fp32 pools are multiplied in fp32.
#include "nxa_paged_units.h"

#include <type_traits>

namespace nxa {

namespace {

constexpr int kStepKeys = 16;

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Step;  // products of one 16-token step

template <>
struct Step<bf16> {
  static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 pv(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                     __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x2 pack(f32x4 x) {
    const bf16x4 r = {(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
    return __builtin_bit_cast(u32x2, r);
  }
  static __device__ __forceinline__ f32x4 unpack(u32x2 x) {
    const bf16x4 r = __builtin_bit_cast(bf16x4, x);
    return f32x4{(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
  }
};
template <>
struct Step<f16> {
  static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 pv(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                 __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x2 pack(f32x4 x) {
    const f16x4 r = {(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3]};
    return __builtin_bit_cast(u32x2, r);
  }
  static __device__ __forceinline__ f32x4 unpack(u32x2 x) {
    const f16x4 r = __builtin_bit_cast(f16x4, x);
    return f32x4{(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
  }
};

// Loads of one step in flight, and how they are consumed.
template <typename T, int DP>
struct StepRegs {
  static constexpr int ES = sizeof(T), CPR = 16 / ES;   // elements of a 16-byte chunk
  static constexpr int NK = DP / (4 * CPR);             // K chunks of a lane
  static constexpr int DPL = DP / 16, NV = DPL * ES / 4;  // V columns, dwords of a lane and key
  u32x4 k[NK];
  Words<NV> v[4];
};

}  // namespace

// Registers: the loads of NB steps (8 KB a wave and step at D = 128, 16 bits)
// beside Q and O; two blocks a CU, one where a step alone is 128 registers.
template <typename T, int DP>
constexpr int kPagedDepth = sizeof(T) * DP <= 256 ? 4 : 2;
template <typename T, int DP>
constexpr int kPagedOcc = DP <= 128 ? 2 : 1;

// P16: pages hold a multiple of 16 tokens, so a step lies in one page and its
// address is uniform; else every key looks its page up.
template <typename T, int DP, bool P16>
__global__ __launch_bounds__(256, (kPagedOcc<T, DP>)) void paged_kernel(const PagedParams p) {
  using R = StepRegs<T, DP>;
  constexpr int ES = R::ES, CPR = R::CPR, NK = R::NK, DPL = R::DPL, NV = R::NV;
  constexpr int NB = kPagedDepth<T, DP>;
  constexpr int NF = DPL;  // O^T fragments: fragment f is columns DPL i + f, i = 0 .. 15
  constexpr bool F32 = std::is_same<T, float>::value;
  constexpr int FIELDS = NF * 4 + 2;
  __shared__ float ms[kWaves * FIELDS * 64];
  __shared__ int pre[257], wsum[kWaves];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int HV = p.Hk * p.strips;

  // The units of this block, u .. u1, numbered from `before` tiles of sequences
  // before b on.
  int64_t u, u1, units = 0;
  int b, before, nblk = 0;
  if (p.nblk == 0) {
    b = blockIdx.x / HV;
    before = 0;
    const int n = paged_units<kStartUnits>(p, b), hv = blockIdx.x % HV;
    if (n == 0) {
      if (hv == 0) paged_zero<T>(p, b);
      return;
    }
    u = (int64_t)hv * n;
    u1 = u + n;
  } else {
    for (int i = blockIdx.x; i < p.B; i += p.nblk)
      if (paged_len(p, i) == 0) paged_zero<T>(p, i);
    if (tid == 0) p.joins[blockIdx.x] = {0, 0, 0, 0};
    paged_prefix<kStartUnits>(p, pre, wsum);
    units = (int64_t)__builtin_amdgcn_readfirstlane(pre[256]) * HV;
    nblk = busy_blocks(p, units);
    if ((int)blockIdx.x >= nblk) return;
    u = first_unit(units, blockIdx.x, nblk);
    u1 = first_unit(units, blockIdx.x + 1, nblk);
    // The sequence of unit u: the last group that starts at or before it, then
    // along the group.
    const int x = (int)(u / HV);
    int lo = 0, hi = 256;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= x) lo = mid;
      else hi = mid;
    }
    b = lo * ((p.B + 255) / 256);
    before = pre[lo];
    for (int n; before + (n = paged_units<kStartUnits>(p, b)) <= x; ++b) before += n;
    b = __builtin_amdgcn_readfirstlane(b);
    before = __builtin_amdgcn_readfirstlane(before);
  }
  const int64_t u0 = u;

  // Per-lane byte offsets inside a step.  K: key c, 16-byte chunk g + 4 j.  V:
  // key 4 g + j, columns DPL c ...  Columns past the head dim are taken from
  // beyond the range: zeros.
  uint32_t koff[NK], voff[4];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    const int d = CPR * (g + 4 * j);
    koff[j] = d < p.D ? (uint32_t)((P16 ? c * p.k_str[2] : 0) + d) * ES : 0xfffffff0u;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    voff[j] = DPL * c < p.Dv ? (uint32_t)((P16 ? (4 * g + j) * p.v_str[2] : 0) + DPL * c) * ES
                             : 0xffffff00u;

  while (u < u1) {
    const int len = __builtin_amdgcn_readfirstlane(paged_len(p, b));
    if (len == 0) {
      ++b;
      continue;
    }
    const int n = paged_tiles(len) + kStartUnits;
    const int64_t rem = u - (int64_t)before * HV;
    const int hv = __builtin_amdgcn_readfirstlane((int)(rem / n));
    const int v0 = __builtin_amdgcn_readfirstlane((int)(rem % n));
    const int v1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)n, v0 + (u1 - u)));
    const int t0 = max(v0 - kStartUnits, 0), t1 = max(v1 - kStartUnits, 0);  // tiles
    const int hk = hv / p.strips, h0 = (hv % p.strips) * 16;
    const int heads = min(16, p.G - h0);

    // Q^T: column c is head h0 + c, chunks as K's.
    u32x4 qf[NK];
    {
      const T* qp = (const T*)p.q + b * p.q_str[0] + ((int64_t)hk * p.G + h0 + min(c, heads - 1)) * p.q_str[1];
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        const int d = CPR * (g + 4 * j);
        qf[j] = c < heads && d < p.D ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{0, 0, 0, 0};
      }
    }
    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_ref = -INFINITY, l = 0.f;

    // This wave's steps: two of the eight of each unit, up to the length.
    const T* kb = (const T*)p.k + hk * p.k_str[1];
    const T* vb = (const T*)p.v + hk * p.v_str[1];
    auto key_of = [&](int i) { return (t0 + (i >> 1)) * kPagedKeys + wave * 32 + (i & 1) * kStepKeys; };
    int steps = 2 * (t1 - t0);
    while (steps > 0 && key_of(steps - 1) >= len) --steps;

    for (int i0 = 0; i0 < steps; i0 += 64) {
      const int ns = min(64, steps - i0);
      // Lane i looks up step i0 + i: its page's and slot's offsets, and the
      // tokens it has (none where the table has no page).
      int64_t kofs = 0, vofs = 0;
      int rows = 0;
      if (P16 && lane < ns) {
        const int key0 = key_of(i0 + lane);
        const int page = p.table[b * p.table_rs + key0 / p.PS], slot = key0 % p.PS;
        if ((unsigned)page < (unsigned)p.P) {
          rows = min(kStepKeys, len - key0);
          kofs = page * p.k_str[0] + slot * p.k_str[2];
          vofs = page * p.v_str[0] + slot * p.v_str[2];
        }
      }
      auto uni64 = [&](int64_t x, int i) -> int64_t {
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, i);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)x >> 32), i);
        return (int64_t)((uint64_t)hi << 32 | lo);
      };
      R ring[NB];
      int have[NB];       // tokens of the step (P16), or a bit a token
      auto issue = [&](int i, R& r, int& hv_rows) NXA_INLINE {
        if constexpr (P16) {
          // (past the last step: empty ranges, so every step counts alike)
          const int j = min(i, ns - 1);
          const int nr = i < ns ? __builtin_amdgcn_readlane(rows, j) : 0;
          const T* ks = kb + uni64(kofs, j);
          const T* vs = vb + uni64(vofs, j);
          const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
              (void*)ks, 0, nr > 0 ? (int)(((nr - 1) * p.k_str[2] + p.D) * ES) : 0, 0x00020000);
          const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
              (void*)vs, 0, nr > 0 ? (int)(((nr - 1) * p.v_str[2] + p.Dv) * ES) : 0, 0x00020000);
#pragma unroll
          for (int x = 0; x < NK; ++x) r.k[x] = __builtin_bit_cast(u32x4, buf_load<4>(rk, koff[x]));
#pragma unroll
          for (int x = 0; x < 4; ++x) r.v[x] = buf_load<NV>(rv, voff[x]);
          hv_rows = nr;
        } else {
          // Lane x < 16 looks up token x of the step; the others ask it.
          const int key = key_of(i0 + min(i, ns - 1)) + c;
          int page = -1;
          if (i < ns && key < len) page = p.table[b * p.table_rs + key / p.PS];
          const bool ok = (unsigned)page < (unsigned)p.P;
          const int64_t kr = ok ? page * p.k_str[0] + (key % p.PS) * p.k_str[2] : 0;
          const int64_t vr = ok ? page * p.v_str[0] + (key % p.PS) * p.v_str[2] : 0;
          hv_rows = (int)(__ballot(ok) & 0xffff);
          const bool kd = ok;
#pragma unroll
          for (int x = 0; x < NK; ++x)
            r.k[x] = kd && koff[x] != 0xfffffff0u
                         ? *reinterpret_cast<const u32x4*>((const char*)(kb + kr) + koff[x])
                         : u32x4{0, 0, 0, 0};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int src = 4 * g + x;
            const int64_t row = (int64_t)((uint64_t)(uint32_t)__shfl((int)((uint64_t)vr >> 32), src, 64) << 32 |
                                          (uint32_t)__shfl((int)(uint32_t)vr, src, 64));
            const bool vok = (hv_rows >> src & 1) && voff[x] != 0xffffff00u;
            const char* at = (const char*)(vb + row) + (vok ? voff[x] : 0u);
            // (of a lane's 16-byte chunks some may lie behind the row's end)
#pragma unroll
            for (int w = 0; w < NV; ++w)
              r.v[x].w[w] = vok && DPL * c + (w & ~3) * (4 / ES) < p.Dv
                                ? reinterpret_cast<const uint32_t*>(at)[w]
                                : 0u;
          }
        }
      };
      auto compute = [&](const R& r, int hv_rows) NXA_INLINE {
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, r.k[j])[e],
                                                       __builtin_bit_cast(f32x4, qf[j])[e], s, 0, 0, 0);
          } else {
            s = Step<T>::qk(r.k[j], qf[j], s);
          }
        }
        // Rows of the accumulator: tokens 4 g + e.
        float mt = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = P16 ? 4 * g + e < hv_rows : (hv_rows >> (4 * g + e) & 1) != 0;
          s[e] = ok ? s[e] * p.scale_log2 : -INFINITY;
          mt = fmaxf(mt, s[e]);
        }
        if (__any(mt > m_ref + kSlack)) {
          mt = fmaxf(mt, xor16(mt));
          mt = fmaxf(mt, shfl_xor32(mt));
          const float mn = fmaxf(m_ref, mt);
          const float alpha = mn > m_ref ? fast_exp2(m_ref - mn) : 1.f;
          l *= alpha;
#pragma unroll
          for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[f][e] *= alpha;
          m_ref = mn;
        }
        const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = fast_exp2(s[e] + neg_m);
        // (l counts the very P that the second product sees)
        l += (s[0] + s[1]) + (s[2] + s[3]);
        if constexpr (F32) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int f = 0; f < NF; ++f)
              o[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, r.v[x].w[f]), s[x],
                                                          o[f], 0, 0, 0);
        } else {
          // P as the sum of two numbers of the I/O type: the matrix core has
          // the time, and P then adds nothing to the output's own rounding.
          const u32x2 pf = Step<T>::pack(s), pl = Step<T>::pack(s - Step<T>::unpack(pf));
#pragma unroll
          for (int w = 0; w < NV; ++w) {
            // Columns 2 w and 2 w + 1 of four keys.
            const u32x2 lo = {__builtin_amdgcn_perm(r.v[1].w[w], r.v[0].w[w], 0x05040100u),
                              __builtin_amdgcn_perm(r.v[3].w[w], r.v[2].w[w], 0x05040100u)};
            const u32x2 hi = {__builtin_amdgcn_perm(r.v[1].w[w], r.v[0].w[w], 0x07060302u),
                              __builtin_amdgcn_perm(r.v[3].w[w], r.v[2].w[w], 0x07060302u)};
            o[2 * w] = Step<T>::pv(lo, pf, o[2 * w]);
            o[2 * w + 1] = Step<T>::pv(hi, pf, o[2 * w + 1]);
            o[2 * w] = Step<T>::pv(lo, pl, o[2 * w]);
            o[2 * w + 1] = Step<T>::pv(hi, pl, o[2 * w + 1]);
          }
        }
      };
#pragma unroll
      for (int x = 0; x < NB; ++x) issue(x, ring[x], have[x]);
      for (int i = 0; i < ns; i += NB)
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          compute(ring[x], have[x]);
          issue(i + x + NB, ring[x], have[x]);
        }
    }
    l += xor16(l);
    l += shfl_xor32(l);

    // Join the waves: [wave][field][lane], field 4 f + e of O, then m and l.
    __syncthreads();
    {
      float* mw = ms + wave * FIELDS * 64 + lane;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) mw[(4 * f + e) * 64] = o[f][e];
      mw[(FIELDS - 2) * 64] = m_ref;
      mw[(FIELDS - 1) * 64] = l;
    }
    __syncthreads();
    {
      float sc[kWaves], mx = -INFINITY, lt = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, ms[(w * FIELDS + FIELDS - 2) * 64 + lane]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float m = ms[(w * FIELDS + FIELDS - 2) * 64 + lane];
        sc[w] = m == -INFINITY ? 0.f : fast_exp2(m - mx);
        lt = __builtin_fmaf(ms[(w * FIELDS + FIELDS - 1) * 64 + lane], sc[w], lt);
      }
      // Wave e takes row e of each fragment: columns DPL (4 g + e) + f.
      const int d0 = DPL * (4 * g + wave);
      float x[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        x[f] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          x[f] = __builtin_fmaf(ms[(w * FIELDS + 4 * f + wave) * 64 + lane], sc[w], x[f]);
      }
      if (v0 == 0 && v1 == n) {
        // (no page of the row valid: no keys, zero)
        const float inv = lt > 0.f || lt != lt ? 1.0f / lt : 0.f;
        if (c < heads && d0 < p.Dv) {
          T* op = (T*)p.o + b * p.o_str[0] + ((int64_t)hk * p.G + h0 + c) * p.o_str[1] + d0;
#pragma unroll
          for (int f = 0; f < NF; ++f)
            if (d0 + f < p.Dv) op[f] = (T)(x[f] * inv);
        }
      } else if (c < heads) {
        const int slot = 2 * blockIdx.x + (u > u0 ? 1 : 0);
        if (v0 == 0 && tid == 0) {
          // The row's last unit is the block j's with first_unit(j) <= it.
          const int64_t z = u + n - 1;
          const int last = (int)(((z + 1) * nblk - 1) / units);
          p.joins[blockIdx.x] = {b, hv, last - (int)blockIdx.x + 1, slot};
        }
        float* part = p.part + (int64_t)slot * paged_part_floats(DP);
#pragma unroll
        for (int f = 0; f < NF; ++f) part[c * DP + d0 + f] = x[f];
        if (wave == 0 && g == 0) {
          part[16 * DP + c] = mx;
          part[16 * DP + 16 + c] = lt;
        }
      }
    }
    u += v1 - v0;
    if (hv == HV - 1 && v1 == n) {
      before += n;
      ++b;
    }
  }
}

// Joins the pieces of the rows that several blocks shared, in the blocks'
// order: block i the row that starts in block i.
template <typename T, int DP>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedParams p) {
  __shared__ float wgt[kJoinPieces * 16];
  __shared__ float inv_s[16];
  __shared__ float acc_s[256 * 4];
  const int tid = threadIdx.x, j0 = blockIdx.x;
  const int4 row = p.joins[j0];
  const int b = row.x, hv = row.y, np = row.z, first = row.w;
  if (np == 0) return;
  const int hk = hv / p.strips, h0 = (hv % p.strips) * 16, heads = min(16, p.G - h0);
  T* op = (T*)p.o + b * p.o_str[0] + ((int64_t)hk * p.G + h0) * p.o_str[1];
  // (the later pieces are their blocks' first results)
  auto piece = [&](int i) {
    return p.part + (int64_t)(i == 0 ? first : 2 * (j0 + i)) * paged_part_floats(DP);
  };
  {
    // 16 threads a head.
    const int h = tid >> 4, sub = tid & 15;
    float m = -INFINITY;
    if (h < heads)
      for (int i = sub; i < np; i += 16) {
        const float x = piece(i)[16 * DP + h];
        wgt[i * 16 + h] = x;
        m = fmaxf(m, x);
      }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) m = fmaxf(m, __shfl_xor(m, d, 64));
    float l = 0.f;
    if (h < heads)
      for (int i = sub; i < np; i += 16) {
        const float x = wgt[i * 16 + h];
        const float w = x == -INFINITY ? 0.f : fast_exp2(x - m);
        wgt[i * 16 + h] = w;
        l = __builtin_fmaf(piece(i)[16 * DP + 16 + h], w, l);
      }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) l += __shfl_xor(l, d, 64);
    if (sub == 0) inv_s[h] = l > 0.f || l != l ? 1.0f / l : 0.f;
  }
  __syncthreads();
  // Four columns a thread; where the row is narrower than the block, groups of
  // threads take every ng-th piece and add up in order.
  const int nv = heads * (DP / 4);
  const int ng = nv >= 256 ? 1 : 256 / nv;
  for (int v0 = 0; v0 < nv; v0 += 256) {
    const int grp = ng > 1 ? tid / nv : 0, v = ng > 1 ? tid % nv : v0 + tid;
    const int h = v / (DP / 4), d = (v % (DP / 4)) * 4;
    const bool on = grp < ng && v < nv;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (on)
#pragma unroll 4
      for (int i = grp; i < np; i += ng) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(piece(i) + h * DP + d);
        const float w = wgt[i * 16 + h];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(y[e], w, x[e]);
      }
    if (ng > 1) {
      *reinterpret_cast<f32x4*>(acc_s + 4 * tid) = x;
      __syncthreads();
      if (grp == 0)
        for (int k = 1; k < ng; ++k) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(acc_s + 4 * (k * nv + tid));
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] += y[e];
        }
    }
    if (on && grp == 0) {
      const float inv = inv_s[h];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < p.Dv) op[h * p.o_str[1] + d + e] = (T)(x[e] * inv);
    }
  }
}

int paged_dp(int m) { return m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256; }

// Rows of up to 1024 tokens gain less from several blocks than the join costs:
// us in a graph, split and whole, head dim 128, 8 heads: one sequence of 256
// 12.5 / 8.0, 1024 12.6 / 14.6 (24.5 / 22.0 with the host's work), 2048 13.6 /
// 31.6; 64 of up to 512 26 / 17, 1024 33 / 27, 2048 47 / 44, 4096 62 / 81; 256 of
// up to 1024 90 / 83, 2048 139 / 138.
bool paged_whole(int64_t room) { return room <= 1024; }

template <typename T, int DP>
static void launch_paged_t(const PagedParams& p, hipStream_t stream) {
  const dim3 grid(p.nblk ? p.nblk : p.B * p.Hk * p.strips), block(256);
  if (p.PS % kStepKeys == 0)
    hipLaunchKernelGGL((paged_kernel<T, DP, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((paged_kernel<T, DP, false>), grid, block, 0, stream, p);
  if (p.nblk)
    hipLaunchKernelGGL((paged_join_kernel<T, DP>), dim3(p.nblk), block, 0, stream, p);
}

template <typename T>
static void launch_paged_d(const PagedParams& p, hipStream_t stream) {
  switch (paged_dp(p.D > p.Dv ? p.D : p.Dv)) {
    case 32: launch_paged_t<T, 32>(p, stream); break;
    case 64: launch_paged_t<T, 64>(p, stream); break;
    case 128: launch_paged_t<T, 128>(p, stream); break;
    default: launch_paged_t<T, 256>(p, stream); break;
  }
}

template <typename T>
static void launch_join_d(const PagedParams& p, int dp, hipStream_t stream) {
  const dim3 grid(p.nblk), block(256);
  switch (dp) {
    case 64: hipLaunchKernelGGL((paged_join_kernel<T, 64>), grid, block, 0, stream, p); break;
    case 128: hipLaunchKernelGGL((paged_join_kernel<T, 128>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((paged_join_kernel<T, 256>), grid, block, 0, stream, p); break;
  }
}

void launch_paged_join(const PagedParams& p, int io_dtype, int dp, hipStream_t stream) {
  if (io_dtype == kF32) launch_join_d<float>(p, dp, stream);
  else if (io_dtype == kF16) launch_join_d<f16>(p, dp, stream);
  else launch_join_d<bf16>(p, dp, stream);
}

void launch_paged(const PagedParams& p, int io_dtype, hipStream_t stream) {
  if (io_dtype == kF32) launch_paged_d<float>(p, stream);
  else if (io_dtype == kF16) launch_paged_d<f16>(p, stream);
  else launch_paged_d<bf16>(p, stream);
}

}  // namespace nxa
