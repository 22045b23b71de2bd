// Attention of one new token a sequence over a quantised paged cache
// (nxa_quant.h): S_j = scale (s_j (q . c_j) + z_j sum q), P = softmax(S) and
// o = sum_j P_j (s'_j c'_j + z'_j), codes c of 4 or 8 bits with a scale and a
// minimum a row.
//
// The pages are never expanded.  Codes enter the matrix products as what they
// are, small whole numbers; the scale of a key multiplies its score behind the
// first product, that of a value its P before the second, and the minima add one
// number a head to the output.  So nothing of a key or value is rounded.  What
// bounds the kernel is what it costs to make operands of codes (1.25 operations a
// code of four bits in a plain form, with the HBM idle two thirds of the time), so
// they are taken as numbers whose bits they already are:
//
//  * K: codes in the mantissa of an fp16 64 (4 bits) or 1024 (8 bits).  What is added
//    to them is what a product's sum starts from, -64 (1024) sum q: a score loses
//    some 2^-24 of s times 64 (1024) |sum q|, eight times what its codes' own sum would.
//    q is scaled to a largest element of 2^14 or more and then is one fp16 number, exact
//    down to 2^-29 of that.  (fp8 numbers need no 64, c 2^-9 being their bits, and three
//    operations for 8 codes in place of seven.  But their products keep 13 bits below
//    the largest of eight and drop the others' rest, and q takes two or three of them.)
//  * V: the same, in pairs of one column's keys.  What is added to the codes would cost
//    digits: the values of a long row nearly cancel, to a root of its length, while
//    their sum with 64 or 1024 does not (65536 tokens of equal weight in bf16 and 4 bits were
//    off by 2.8e-2 of the output, 1.8e-3 now, its own rounding).  So it comes off every
//    four steps, with the codes' middle, by a product of ones with the very P s' that the
//    other products saw; the rest of a value is s 8 + z (s 128 + z).  P s' is two fp16
//    numbers (off by 2^-23; one, in bf16, would take 2 us of 49 less and be off by
//    2^-12), times a power of two that keeps the largest of them near the top of
//    fp16's range.
//  * fp32: four steps' sums of 64s would cost digits too.  So K's and V's codes are fp16
//    numbers from -8 or -128 on, one packed addition more, what they are counted from is
//    (s 8 + z) or (s 128 + z), and q and P s' are three fp16 numbers each.
//
// The blocks share the work as in nxa_paged.hip (units of 128 tokens, pieces of
// a row joined by its second kernel).  A step of a wave is 32 tokens, two halves
// of 16: S^T = K Q^T a half, whose accumulator holds P^T as the second product reads
// it, O^T += V^T P^T over all 32.  Per half a lane takes a quarter of one key's
// codes (the head dim of a product is summed in any order, so q is read in the
// order of the codes), DP / 16 columns of four keys' values, and the scales of those
// four keys.
//
// At head dim 128 and 8 key heads, kernel without the join: two sequences, 582,048
// tokens together, in 4 bits (633 MB) 116 us, 5.5 TB/s, nine tenths of the rate of
// reading alone; 64 of up to 8192 (154 MB) 47 us, of which starting on rows and the
// first copies' latency are some 15; in 8 bits (351 MB) 75 us, 4.7 TB/s.
#include "nxa_quant.h"

#include "nxa_paged_units.h"

#include <type_traits>

namespace nxa {

namespace {

constexpr int kHalfKeys = 16;

template <typename T, int DP, int BITS>
struct QuantStep {
  static constexpr int ES = sizeof(T);
  static constexpr bool F32 = ES == 4;
  static constexpr int NKW = DP * BITS / 128;       // dwords of K's codes a lane and half
  static constexpr int NJ = DP / 32;                // products of a half's S
  static constexpr int DPL = DP / 16;               // V columns of a lane
  static constexpr int VB = DPL * BITS / 8;         // bytes of them a key
  static constexpr int NVW = VB >= 4 ? VB / 4 : 1;  // dwords
  static constexpr int NS = ES;                     // dwords of a token's scales: 4 ES / 4
  static constexpr int QT = F32 ? 3 : 1;            // terms of q
  static constexpr int PT = F32 ? 3 : 2;            // of P s'
  static constexpr float MID = BITS == 4 ? 8.f : 128.f;     // V's codes count from it (fp32: K's too)
  static constexpr float ZERO = BITS == 4 ? 64.f : 1024.f;  // what stands in for 0 (16-bit types)
  // A half in LDS: K's codes, V's, the scales; copies of 1 KB (scales: 256 bytes).
  static constexpr int KC = DP * BITS <= 512 ? 1 : DP * BITS / 512;
  static constexpr int HALF_BYTES = 2 * 1024 * KC + 256;
  static constexpr int COPIES = 2 * KC + 1;
};

// N dwords of a lane.
template <int N>
struct Loaded {
  uint32_t w[N];
  __device__ __forceinline__ uint32_t at(int i) const { return w[i]; }
  // From LDS (aligned to what is read, up to 16 bytes).
  __device__ __forceinline__ void lds(uint32_t at) {
    constexpr int W = N < 4 ? N : 4;
    typedef uint32_t V __attribute__((ext_vector_type(W)));
    typedef __attribute__((address_space(3))) const V lds_v;
#pragma unroll
    for (int i = 0; i < N; i += W) {
      const V x = *(lds_v*)(uintptr_t)(at + 4 * i);
#pragma unroll
      for (int j = 0; j < W; ++j) w[i + j] = x[j];
    }
  }
};

// A half's codes and scales of a lane.
template <typename T, int DP, int BITS>
struct HalfRegs {
  using R = QuantStep<T, DP, BITS>;
  Loaded<R::NKW> k;
  Loaded<R::NVW> v[4];
  Loaded<R::NS> s[4];
};

__device__ __forceinline__ f32x4 mma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// Two numbers as fp16, the first in the low half.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 r = {(f16)a, (f16)b};
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float low_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float low_f16(uint32_t w) {
  return (float)__builtin_bit_cast(f16, (uint16_t)w);
}
__device__ __forceinline__ float high_f16(uint32_t w) {
  return (float)__builtin_bit_cast(f16, (uint16_t)(w >> 16));
}

// Constants of the codes' masks, kept in registers of both kinds, so that an and
// and an or are one operation (two constants of it cannot both be literals).
struct CodeBits {
  uint32_t high, k1024, k64, from64, from1024;
  __device__ __forceinline__ CodeBits() {
    asm("s_mov_b32 %0, 0x00f000f0" : "=s"(high));
    asm("v_mov_b32 %0, 0x64006400" : "=v"(k1024));
    asm("v_mov_b32 %0, 0x54005400" : "=v"(k64));
    asm("s_mov_b32 %0, 0xd480d480" : "=s"(from64));    // -(64 + 8) twice, as fp16
    asm("s_mov_b32 %0, 0xe480e480" : "=s"(from1024));  // -(1024 + 128)
  }
};

// Two fp16 sums.
__device__ __forceinline__ uint32_t add_f16(uint32_t a, uint32_t b) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) + __builtin_bit_cast(f16x2, b));
}
// The nibbles at bits SH .. SH + 3 and SH + 16 .. SH + 19 as fp16, more by 64.
template <int SH>
__device__ __forceinline__ uint32_t nibbles_f16(uint32_t w, const CodeBits& cb) {
  return ((SH < 4 ? w << (4 - SH) : w >> (SH - 4)) & cb.high) | cb.k64;
}
// Two bytes (of a word, as `sel` picks them into the low ones), more by 1024.
__device__ __forceinline__ uint32_t bytes_f16(uint32_t w, uint32_t sel, const CodeBits& cb) {
  return __builtin_amdgcn_perm(0u, w, sel) | cb.k1024;
}
// Product operand j of a lane's codes of one key, eight of them; MID: from their
// middle, else more by what stands in for 0.
template <int BITS, bool MID, int N>
__device__ __forceinline__ u32x4 key_f16(const Loaded<N>& k, int j, const CodeBits& cb) {
  u32x4 r;
  if constexpr (BITS == 4) {
    const uint32_t w = k.at(j);
    r = u32x4{nibbles_f16<0>(w, cb), nibbles_f16<4>(w, cb), nibbles_f16<8>(w, cb),
              nibbles_f16<12>(w, cb)};
  } else {
    const uint32_t a = k.at(2 * j), b = k.at(2 * j + 1);
    r = u32x4{bytes_f16(a, 0x0c010c00u, cb), bytes_f16(a, 0x0c030c02u, cb),
              bytes_f16(b, 0x0c010c00u, cb), bytes_f16(b, 0x0c030c02u, cb)};
  }
  if constexpr (MID)
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = add_f16(r[i], BITS == 4 ? cb.from64 : cb.from1024);
  return r;
}
// The element of eight that stands at place e of an operand.
template <int BITS>
__device__ constexpr int key_order(int e) {
  return BITS == 8 ? e : (e >> 1) + 4 * (e & 1);
}

// The lane eight columns on (of sixteen).
__device__ __forceinline__ uint32_t other_eight(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true);
}
__device__ __forceinline__ float other_eight(float x) {
  return __uint_as_float(other_eight(__float_as_uint(x)));
}

// What the middle of a row's codes stands for.
template <typename T, int BITS>
__device__ __forceinline__ float from_mid(float s, float z) {
  return __builtin_fmaf(s, QuantStep<T, 16, BITS>::MID, z);
}
// Scales of a token: fields k's scale and minimum, v's.
template <typename T, int N>
__device__ __forceinline__ float scale_field(const Loaded<N>& s, int f) {
  if constexpr (std::is_same<T, float>::value)
    return __uint_as_float(s.at(f));
  else if constexpr (std::is_same<T, f16>::value)
    return f & 1 ? high_f16(s.at(f >> 1)) : low_f16(s.at(f >> 1));
  else
    return f & 1 ? high_of(s.at(f >> 1)) : low_of(s.at(f >> 1));
}

}  // namespace

// Steps whose copies are in flight.
constexpr int kQuantDepth = 2;
// Blocks a CU, by registers and LDS (37 KB at 512 bits a row and less, 70 KB at
// 1024): three where q and O leave room for it (64 sequences of up to 8192, 4 bits,
// three / two: 53.6 / 57.0 us a call; more than eight heads a key head, where three
// spill 12 registers, 93 / 107).
constexpr int quant_blocks(int es, int dp, int bits) {
  return dp > 128 ? 1 : dp * bits > 512 || (es == 4 && dp == 128) ? 2 : 3;
}

// FAST: pages hold a multiple of 16 tokens, so that a half lies in one page, and
// codes and scales are aligned: halves are copied to LDS, each wave its own, steps
// ahead of their use.  Else every key looks its page up and codes are loaded four
// bytes at a time (64 sequences of up to 8192, 4 bits, 54 / 79 us, 8 bits 73 / 162).
// PAIR: eight heads a key head or fewer leave half of a product's columns idle.  q
// then stands in both halves, and columns from 8 on take the softmax of the second
// half's keys, whose weights go back to the heads' columns for V's product (two
// sequences of up to 400000, four heads a key head, with / without 130 / 146 us).
template <typename T, int DP, int BITS, bool FAST, bool PAIR>
__global__ __launch_bounds__(256, quant_blocks(sizeof(T), DP, BITS)) void
qpaged_kernel(const QuantPagedParams p) {
  using R = QuantStep<T, DP, BITS>;
  using Half = HalfRegs<T, DP, BITS>;
  constexpr int NKW = R::NKW, NJ = R::NJ, DPL = R::DPL, VB = R::VB, NVW = R::NVW, NS = R::NS;
  constexpr int QT = R::QT, PT = R::PT;
  constexpr int NB = kQuantDepth;
  constexpr int SC = PAIR ? 4 : 8;  // scores of a lane and step
  constexpr int NF = DPL;  // O^T fragments: fragment f is columns DPL i + f, i = 0 .. 15
  constexpr int FIELDS = NF * 4 + 2;
  constexpr int STEP_BYTES = 2 * R::HALF_BYTES, COPIES = R::COPIES;
  constexpr int RING = FAST ? kWaves * NB * STEP_BYTES : 0, JOIN = kWaves * FIELDS * 64 * 4;
  // (the waves' rings, then what they join)
  __shared__ __attribute__((aligned(16))) char mem[RING > JOIN ? RING : JOIN];
  __shared__ int pre[257], wsum[kWaves];
  float* const ms = reinterpret_cast<float*>(mem);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const bool upper = c >= 8;
  const int HV = p.Hk * p.strips;

  // The units of this block, u .. u1 (as in paged_kernel).
  int64_t u, u1, units = 0;
  int b, before, nblk = 0;
  if (p.nblk == 0) {
    b = blockIdx.x / HV;
    before = 0;
    const int n = paged_units<kQuantStart>(p, b), hv = blockIdx.x % HV;
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
    paged_prefix<kQuantStart>(p, pre, wsum);
    units = (int64_t)__builtin_amdgcn_readfirstlane(pre[256]) * HV;
    nblk = busy_blocks(p, units);
    if ((int)blockIdx.x >= nblk) return;
    u = first_unit(units, blockIdx.x, nblk);
    u1 = first_unit(units, blockIdx.x + 1, nblk);
    const int x = (int)(u / HV);
    int lo = 0, hi = 256;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= x) lo = mid;
      else hi = mid;
    }
    b = lo * ((p.B + 255) / 256);
    before = pre[lo];
    for (int n; before + (n = paged_units<kQuantStart>(p, b)) <= x; ++b) before += n;
    b = __builtin_amdgcn_readfirstlane(b);
    before = __builtin_amdgcn_readfirstlane(before);
  }
  const int64_t u0 = u;
  const CodeBits cb;

  // Bytes of a row.  A half in LDS: key c, chunk g of K; columns DPL c .. of V and
  // the scales of keys 4 g ...
  const int kb = p.D * BITS / 8, vb = p.Dv * BITS / 8;
  const uint32_t ring = lds_offset(mem) + wave * (NB * STEP_BYTES);
  const uint32_t k_at = ring + c * kb + 4 * NKW * g;
  const uint32_t v_at = ring + 1024 * R::KC + 4 * g * vb + VB * c;
  const uint32_t s_at = ring + 2048 * R::KC + 16 * R::ES * g + (PAIR && upper ? R::HALF_BYTES : 0);
  typedef const __attribute__((address_space(4))) int constant_int;
  // Pages and slots that 128 tokens span.
  const int per = p.PS >= kPagedKeys ? 0 : kPagedKeys / p.PS, rest = kPagedKeys - per * p.PS;

  while (u < u1) {
    const int len = __builtin_amdgcn_readfirstlane(paged_len(p, b));
    if (len == 0) {
      ++b;
      continue;
    }
    const int n = paged_tiles(len) + kQuantStart;
    const int64_t rem = u - (int64_t)before * HV;
    const int hv = __builtin_amdgcn_readfirstlane((int)(rem / n));
    const int v0 = __builtin_amdgcn_readfirstlane((int)(rem % n));
    const int v1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)n, v0 + (u1 - u)));
    const int t0 = max(v0 - kQuantStart, 0), t1 = max(v1 - kQuantStart, 0);  // tiles
    const int hk = hv / p.strips, h0 = (hv % p.strips) * 16;
    const int heads = min(16, p.G - h0);

    const char* kp = (const char*)p.k + hk * p.k_str[1];
    const char* vp = (const char*)p.v + hk * p.v_str[1];
    const char* sp = (const char*)p.sc + hk * p.sc_str[1] * R::ES;
    // This wave's steps: 32 tokens of each unit, up to the length.
    auto key_of = [&](int half) { return (t0 + (half >> 1)) * kPagedKeys + wave * 32 + (half & 1) * kHalfKeys; };
    int steps = t1 - t0;
    while (steps > 0 && key_of(2 * steps - 2) >= len) --steps;
    // Column and slot of the next half to be issued, and its page (read a half
    // ahead).
    int half = 0, col = 0, slot = 0, page = -1, have[NB][2];
    const auto* row = (constant_int*)(uintptr_t)(p.table + b * p.table_rs);
    if constexpr (FAST) {
      const int key0 = key_of(0);
      col = __builtin_amdgcn_readfirstlane(key0 / p.PS);
      slot = __builtin_amdgcn_readfirstlane(key0 - key0 / p.PS * p.PS);
      page = steps > 0 ? row[col] : -1;
    }
    auto issue = [&](uint32_t to, int& mine) NXA_INLINE {
      // (past the last step: empty ranges, so that every step counts alike)
      const int key0 = key_of(half);
      const bool ok = half < 2 * steps && (unsigned)page < (unsigned)p.P;
      mine = ok ? max(min(kHalfKeys, len - key0), 0) : 0;
      const uint64_t pg = ok ? (uint32_t)page : 0u;
      const uint64_t sl = ok ? (uint32_t)slot : 0u;  // (times a row's bytes: past 32 bits)
      const char* ks = kp + pg * (uint32_t)p.k16 * 16 + sl * (uint32_t)kb;
      const char* vs = vp + pg * (uint32_t)p.v16 * 16 + sl * (uint32_t)vb;
      const char* ss = sp + pg * (uint32_t)p.s16 * 16 + sl * (4 * R::ES);
      // The next half: in this step, or at the same place 128 tokens on.
      ++half;
      if (half & 1) {
        slot += kHalfKeys;
      } else {
        slot += rest - kHalfKeys;
        col += per;
        if (slot < 0) slot += p.PS, --col;
      }
      if (slot >= p.PS) slot -= p.PS, ++col;
      page = half < 2 * steps && key_of(half) < len ? row[col] : -1;
      const i32x4 rk = make_rsrc(ks, mine * kb), rv = make_rsrc(vs, mine * vb),
                  rs = make_rsrc(ss, mine * (4 * R::ES));
#pragma unroll
      for (int x = 0; x < R::KC; ++x) {
        dma16_buf_nt(rk, 16 * lane + 1024 * x, to + 1024 * x);
        dma16_buf_nt(rv, 16 * lane + 1024 * x, to + 1024 * (R::KC + x));
      }
      dma4_buf(rs, 4 * lane, to + 2048 * R::KC);
    };
    auto fetch_v = [&](Half& r, uint32_t at) NXA_INLINE {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if constexpr (VB == 2)
          r.v[x].w[0] = *(const __attribute__((address_space(3))) uint16_t*)(uintptr_t)(v_at + at + x * vb);
        else
          r.v[x].lds(v_at + at + x * vb);
      }
    };
    // (the first copies are on their way while q is read and taken apart)
    if constexpr (FAST)
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) issue(ring + x * STEP_BYTES + h * R::HALF_BYTES, have[x][h]);
    // Q^T: column c is head h0 + c; the lane's quarter of the head dim in the
    // order of K's codes, as QT terms, and the sum of the whole row.
    u32x4 qb[NJ][QT];
    float qsum = 0.f, sl;
    {
      const int cq = PAIR ? c & 7 : c;
      const T* qp = (const T*)p.q + b * p.q_str[0] + ((int64_t)hk * p.G + h0 + min(cq, heads - 1)) * p.q_str[1];
      float x[DP / 4], most = 0.f;
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) {
        const int d = g * (DP / 4) + 8 * j;
        float* y = x + 8 * j;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.f;
        if (cq < heads && d < p.D) {
          const u32x4* src = reinterpret_cast<const u32x4*>(qp + d);
          if constexpr (sizeof(T) == 4) {
            const f32x4 lo = __builtin_bit_cast(f32x4, src[0]), hi = __builtin_bit_cast(f32x4, src[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = lo[e], y[4 + e] = hi[e];
          } else {
            struct alignas(16) Row { T x[8]; };
            const Row r = __builtin_bit_cast(Row, src[0]);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (float)r.x[e];
          }
        }
        // (a negative scale turns q instead, so that the largest score is that of
        // the largest product)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = p.scale_log2 < 0.f ? -y[e] : y[e];
          most = fmaxf(most, __builtin_fabsf(y[e]));
        }
      }
      most = fmaxf(most, xor16(most));
      most = fmaxf(most, shfl_xor32(most));
      // q times 2^up, its largest element in 2^14 .. 2^15: as fp16 exact down to 2^-29
      // of that (16-bit types), in three terms to 2^-24 of each element and 2^-39 of the
      // largest (fp32).  Scores in units of 2^-up.  NaN and infinity of q leave NaN.
      const int up = min(15 - __builtin_amdgcn_frexp_expf(most), 100);
      const float by = most > 0.f ? __builtin_ldexpf(1.f, up) : 1.f;
#pragma unroll
      for (int e = 0; e < DP / 4; ++e) {
        x[e] *= by;
        qsum += x[e];
      }
      qsum += xor16(qsum);
      qsum += shfl_xor32(qsum);
      qsum += (most - most) + (qsum - qsum);
      sl = __builtin_fabsf(p.scale_log2) / by;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float& a = x[8 * j + key_order<BITS>(2 * w)];
            float& o = x[8 * j + key_order<BITS>(2 * w + 1)];
            const uint32_t r = pack_f16(a, o);
            qb[j][t][w] = r;
            a -= low_f16(r), o -= high_f16(r);
          }
      // (one of zero is so small that all scores are zero, but for the -inf of a
      // token that takes no part)
      sl = fmaxf(sl, 0x1p-126f);
    }
    f32x4 o[NF], ones_o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    // P is 2^(score - m_ref): m_ref is the largest score seen, rounded up so that it
    // moves by whole powers of two, and raised by more than 2^kSlack only.  l sums P, zs
    // what the minima add to every column.  P s' goes to fp16 times 2^x_exp, whose
    // range is short: the exponent follows the largest P s' itself, which then is in 2^9
    // .. 2^15 (rows of large scales and no weight do not count), up to 2^kMostExp, past
    // which P 2^x_exp would leave fp32.
    constexpr float kMostExp = 100.f;
    float m_ref = -INFINITY, neg_m = 0.f, l = 0.f, zs = 0.f, x_exp = kMostExp, x_by = 0x1p100f;
    // (over the lanes of a head)
    auto most_of = [&](float x) NXA_INLINE {
      x = fmaxf(x, xor16(x));
      x = fmaxf(x, shfl_xor32(x));
      if constexpr (PAIR) x = fmaxf(x, other_eight(x));
      return x;
    };
    // 2^e of a whole number e at most 0, however small.
    auto shrink = [](float e) NXA_INLINE { return __builtin_ldexpf(1.f, (int)fmaxf(e, -200.f)); };

    // `mine`: tokens of the half (FAST), or a bit a token.
    constexpr int kFull = FAST ? kHalfKeys : 0xffff;
    // (`values` is called between the softmax and V's product)
    auto compute = [&](Half (&r)[2], const int (&mine)[2], auto&& values) NXA_INLINE {
      f32x4 dots[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // (what stands in for 0 in the codes is taken off to begin with)
        const float from = R::F32 ? 0.f : -R::ZERO * qsum;
        dots[h] = f32x4{from, from, from, from};
        f32x4 rest = {0.f, 0.f, 0.f, 0.f};  // fp32: of all terms of q but the first
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const u32x4 a = key_f16<BITS, R::F32>(r[h].k, j, cb);
#pragma unroll
          for (int t = 1; t < QT; ++t) rest = mma_f16(a, qb[j][t], rest);
          dots[h] = mma_f16(a, qb[j][0], dots[h]);
        }
        if constexpr (R::F32)
#pragma unroll
          for (int e = 0; e < 4; ++e) dots[h][e] += rest[e];
      }
      // Rows of the accumulator: tokens 4 g + e.
      float s[SC], vs[SC], vz[SC];
#pragma unroll
      for (int i = 0; i < SC; ++i) {
        const auto& sc = r[i / 4].s[i % 4];
        // (a scale of infinity makes its token NaN, whatever the signs)
        const float ks = scale_field<T>(sc, 0);
        const float z = scale_field<T>(sc, 1), kz = R::F32 ? from_mid<T, BITS>(ks, z) : z;
        const float dot = PAIR && upper ? dots[1][i % 4] : dots[i / 4][i % 4];
        s[i] = __builtin_fmaf(dot, ks, __builtin_fmaf(kz, qsum, ks * 0.f));
        vs[i] = scale_field<T>(sc, 2);
        vz[i] = from_mid<T, BITS>(vs[i], scale_field<T>(sc, 3));
      }
      if (__builtin_expect(((mine[0] ^ kFull) | (mine[1] ^ kFull)) != 0, 0)) {
#pragma unroll
        for (int i = 0; i < SC; ++i) {
          const int e = i % 4, there = PAIR && upper ? mine[1] : mine[i / 4];
          const bool ok = FAST ? 4 * g + e < there : (there >> (4 * g + e) & 1) != 0;
          // (what stands there of other tokens' scales may be NaN)
          s[i] = ok ? s[i] : -INFINITY;
          vs[i] = ok ? vs[i] : 0.f;
          vz[i] = ok ? vz[i] : 0.f;
        }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int i = 0; i < SC; ++i) mt = fmaxf(mt, s[i]);
      mt *= sl;
      float o_by = 1.f;
      if (__builtin_expect(__any(mt > m_ref + kSlack), 0)) {
        const float old = m_ref;
        m_ref = fmaxf(m_ref, __builtin_ceilf(most_of(mt)));
        neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
        // (from -inf on, where nothing has been summed: by 0)
        const float up = m_ref > old ? m_ref - old : 0.f, alpha = shrink(-up);
        l *= alpha;
        zs *= alpha;
        // P s' keeps its power of two, what P loses x_exp gains.
        x_exp += up;
        o_by = shrink(fminf(kMostExp - x_exp, 0.f));
        x_exp = fminf(x_exp, kMostExp);
        x_by = __builtin_ldexpf(1.f, (int)x_exp);
      }
      float w[SC], x[SC], xm = 0.f;  // P and P s'
#pragma unroll
      for (int i = 0; i < SC; ++i) {
        w[i] = fast_exp2(__builtin_fmaf(s[i], sl, neg_m));
        l += w[i];
        zs = __builtin_fmaf(w[i], vz[i], zs);
        x[i] = w[i] * x_by * vs[i];
        xm = fmaxf(xm, __builtin_fabsf(x[i]));
      }
      if (__builtin_expect(__any((xm > 0x1p15f) | (o_by < 1.f)), 0)) {
        float e = -1000.f;
#pragma unroll
        for (int i = 0; i < SC; ++i)
          if (x[i] != 0.f)
            e = fmaxf(e, (float)(__builtin_amdgcn_frexp_expf(w[i]) + __builtin_amdgcn_frexp_expf(vs[i])));
        // (the largest P s' is then in 2^9 .. 2^11)
        const float to = fminf(x_exp, 11.f - most_of(e));
        o_by *= shrink(to - x_exp);
#pragma unroll
        for (int e = 0; e < 4; ++e) ones_o[e] *= o_by;
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[f][e] *= o_by;
        x_exp = to;
        x_by = __builtin_ldexpf(1.f, (int)x_exp);
#pragma unroll
        for (int i = 0; i < SC; ++i) x[i] = w[i] * x_by * vs[i];
      }
      // (a term is to be that of the rounded product, which the next is taken from;
      // the compiler would round the exact one to fp16 for it)
#pragma unroll
      for (int i = 0; i < SC; ++i) asm("" : "+v"(x[i]));
      u32x4 pf[PT];
#pragma unroll
      for (int t = 0; t < PT; ++t)
#pragma unroll
        for (int w = 0; w < SC / 2; ++w) {
          pf[t][w] = pack_f16(x[2 * w], x[2 * w + 1]);
          if constexpr (PAIR) pf[t][2 + w] = other_eight(pf[t][w]);
          x[2 * w] -= low_f16(pf[t][w]);
          x[2 * w + 1] -= high_f16(pf[t][w]);
        }
      values();
      auto product = [&](f32x4& acc, u32x4 a) NXA_INLINE {
#pragma unroll
        for (int t = 0; t < PT; ++t) acc = mma_f16(a, pf[t], acc);
      };
      if constexpr (!R::F32) product(ones_o, u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u});
#pragma unroll
      for (int w = 0; w < NVW; ++w)
#pragma unroll
        for (int y = 0; y < (VB < 4 ? VB : 4); ++y) {
          // Byte y of word w of the lane's eight keys, in pairs.
          const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + y) << 16 | (uint32_t)y;
          u32x4 t, a, d;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            t[i] = __builtin_amdgcn_perm(r[i / 2].v[2 * (i % 2) + 1].at(w), r[i / 2].v[2 * (i % 2)].at(w), sel);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (BITS == 8) {
              a[i] = t[i] | cb.k1024;
              if constexpr (R::F32) a[i] = add_f16(a[i], cb.from1024);
            } else {
              a[i] = (t[i] << 4 & cb.high) | cb.k64;
              d[i] = (t[i] & cb.high) | cb.k64;
              if constexpr (R::F32) a[i] = add_f16(a[i], cb.from64), d[i] = add_f16(d[i], cb.from64);
            }
          }
          if constexpr (BITS == 8) {
            product(o[4 * w + y], a);
          } else {
            product(o[8 * w + 2 * y], a);
            product(o[8 * w + 2 * y + 1], d);
          }
        }
    };
    // What stands in for 0 and the codes' middle off O (16-bit types): before every
    // fourth step, so that the sums stay as small as the values they are made of.
    auto settle = [&]() NXA_INLINE {
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[f][e] = __builtin_fmaf(-(R::ZERO + R::MID), ones_o[e], o[f][e]);
      ones_o = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    if constexpr (FAST) {
      for (int i = 0; i < steps; i += NB) {
        if (!R::F32 && i % 4 == 0) settle();
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          // (the copies of the steps behind it may be in flight)
          __builtin_amdgcn_s_waitcnt(vmcnt_imm((NB - 1) * 2 * COPIES));
          asm volatile("" ::: "memory");
          Half r[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t at = x * STEP_BYTES + h * R::HALF_BYTES;
            r[h].k.lds(k_at + at);
#pragma unroll
            for (int y = 0; y < (PAIR && h ? 0 : 4); ++y) r[h].s[y].lds(s_at + at + 4 * R::ES * y);
          }
          const int mine[2] = {have[x][0], have[x][1]};
          compute(r, mine, [&]() NXA_INLINE {
#pragma unroll
            for (int h = 0; h < 2; ++h) fetch_v(r[h], x * STEP_BYTES + h * R::HALF_BYTES);
            // (all is read before the next copies to this place)
            __builtin_amdgcn_s_waitcnt(lgkmcnt_imm(0));
            asm volatile("" ::: "memory");
#pragma unroll
            for (int h = 0; h < 2; ++h) issue(ring + x * STEP_BYTES + h * R::HALF_BYTES, have[x][h]);
          });
        }
      }
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    } else {
      for (int i = 0; i < steps; ++i) {
        if (!R::F32 && i % 4 == 0) settle();
        Half r[2];
        int mine[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // Lane x < 16 looks up token x of the half; the others ask it.
          const int key = key_of(2 * i + h) + c;
          int page = -1, slot = 0;
          if (key < len) {
            page = p.table[b * p.table_rs + key / p.PS];
            slot = key % p.PS;
          }
          const bool ok = (unsigned)page < (unsigned)p.P;
          if (!ok) page = slot = 0;
          mine[h] = (int)(__ballot(ok) & 0xffff);
          const char* kr = kp + page * p.k_str[0] + (int64_t)slot * kb + 4 * NKW * g;
#pragma unroll
          for (int w = 0; w < NKW; ++w)
            r[h].k.w[w] = ok && 4 * (NKW * g + w) < kb ? reinterpret_cast<const uint32_t*>(kr)[w] : 0u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int src = 4 * g + x;
            const bool on = mine[h] >> src & 1;
            const int64_t vpg = __shfl(page, src, 64), vsl = __shfl(slot, src, 64);
            const char* vr = vp + vpg * p.v_str[0] + vsl * vb + VB * c;
            if constexpr (VB == 2) {
              r[h].v[x].w[0] = on && VB * c < vb ? *reinterpret_cast<const uint16_t*>(vr) : 0u;
            } else {
#pragma unroll
              for (int w = 0; w < NVW; ++w)
                r[h].v[x].w[w] = on && VB * c + 4 * w < vb ? reinterpret_cast<const uint32_t*>(vr)[w] : 0u;
            }
            const uint32_t* sr = reinterpret_cast<const uint32_t*>(
                sp + vpg * p.sc_str[0] * R::ES + vsl * (4 * R::ES));
#pragma unroll
            for (int w = 0; w < NS; ++w) r[h].s[x].w[w] = on ? sr[w] : 0u;
          }
        }
        compute(r, mine, [] {});
      }
    }
    if constexpr (!R::F32) settle();
    l += xor16(l);
    l += shfl_xor32(l);
    zs += xor16(zs);
    zs += shfl_xor32(zs);
    if constexpr (PAIR) {
      l += other_eight(l);
      zs += other_eight(zs);
    }

    // Join the waves: [wave][field][lane], field 4 f + e of O, then m and l (where
    // the rings were: all copies have landed and been read).
    __syncthreads();
    {
      float* mw = ms + wave * FIELDS * 64 + lane;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mw[(4 * f + e) * 64] = __builtin_ldexpf(o[f][e], -(int)x_exp) + zs;
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
        const int piece = 2 * blockIdx.x + (u > u0 ? 1 : 0);
        if (v0 == 0 && tid == 0) {
          // The row's last unit is the block j's with first_unit(j) <= it.
          const int64_t z = u + n - 1;
          const int last = (int)(((z + 1) * nblk - 1) / units);
          p.joins[blockIdx.x] = {b, hv, last - (int)blockIdx.x + 1, piece};
        }
        float* part = p.part + (int64_t)piece * paged_part_floats(DP);
#pragma unroll
        for (int f = 0; f < NF; ++f) part[c * DP + d0 + f] = x[f];
        if (wave == 0 && g == 0) {
          part[16 * DP + c] = mx;
          part[16 * DP + 16 + c] = lt;
        }
      }
    }
    if constexpr (FAST) __syncthreads();  // (the next row's copies)
    u += v1 - v0;
    if (hv == HV - 1 && v1 == n) {
      before += n;
      ++b;
    }
  }
}

int qpaged_dp(int m) { return m <= 64 ? 64 : m <= 128 ? 128 : 256; }

// Rows a block each, of tables this short, against rows cut into equal work and
// joined.  us a call at head dim 128, 4 bits: 32 rows of 700 or 1000 tokens 18 / 23, of
// 2000 25.3 / 22.8; 256 rows of up to 2048 25.6 / 30.3, 512 33.4 / 38.6; 512 of up to
// 4096 54 / 48.
bool qpaged_whole(int64_t room, int64_t rows) {
  return room <= (rows < 256 ? 1024 : 2304);
}

int qpaged_blocks(int io_dtype, int dp, int bits) {
  return 256 * (dp > 128 ? 2 : quant_blocks(io_dtype == kF32 ? 4 : 2, dp, bits));
}

template <typename T, int DP, int BITS>
static void launch_qpaged_b(QuantPagedParams p, hipStream_t stream) {
  const dim3 grid(p.nblk ? p.nblk : p.B * p.Hk * p.strips), block(256);
  using R = QuantStep<T, DP, BITS>;
  const int kb = p.D * BITS / 8, vb = p.Dv * BITS / 8;
  const int64_t ps = p.sc_str[0] * (int)sizeof(T), hs = p.sc_str[1] * (int)sizeof(T);
  const bool aligned = !((p.k_str[0] | p.k_str[1] | p.v_str[0] | p.v_str[1] | ps | hs) & 15);
  const int64_t far = (int64_t)1 << 35;  // (a page stride counts 16 bytes in 31 bits)
  if (p.PS % kHalfKeys == 0 && kb % (4 * R::NKW) == 0 && vb % R::VB == 0 && aligned &&
      p.k_str[0] < far && p.v_str[0] < far && ps < far) {
    p.k16 = (int)(p.k_str[0] / 16);
    p.v16 = (int)(p.v_str[0] / 16);
    p.s16 = (int)(ps / 16);
    if (p.G <= 8)
      hipLaunchKernelGGL((qpaged_kernel<T, DP, BITS, true, true>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((qpaged_kernel<T, DP, BITS, true, false>), grid, block, 0, stream, p);
  } else {
    hipLaunchKernelGGL((qpaged_kernel<T, DP, BITS, false, false>), grid, block, 0, stream, p);
  }
}

template <typename T, int BITS>
static void launch_qpaged_d(const QuantPagedParams& p, hipStream_t stream) {
  switch (qpaged_dp(p.D > p.Dv ? p.D : p.Dv)) {
    case 64: launch_qpaged_b<T, 64, BITS>(p, stream); break;
    case 128: launch_qpaged_b<T, 128, BITS>(p, stream); break;
    default: launch_qpaged_b<T, 256, BITS>(p, stream); break;
  }
}

template <typename T>
static void launch_qpaged_t(const QuantPagedParams& p, hipStream_t stream) {
  if (p.bits == 4) launch_qpaged_d<T, 4>(p, stream);
  else launch_qpaged_d<T, 8>(p, stream);
}

void launch_quant_paged(const QuantPagedParams& p, int io_dtype, hipStream_t stream) {
  if (io_dtype == kF32) launch_qpaged_t<float>(p, stream);
  else if (io_dtype == kF16) launch_qpaged_t<f16>(p, stream);
  else launch_qpaged_t<bf16>(p, stream);
  if (p.nblk) launch_paged_join(p, io_dtype, qpaged_dp(p.D > p.Dv ? p.D : p.Dv), stream);
}

}  // namespace nxa
