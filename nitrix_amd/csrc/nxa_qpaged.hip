// Attention of one new token a sequence over a quantised paged cache
// (nxa_quant.h): S_j = scale (s_j (q . c_j) + z_j sum q), P = softmax(S) and
// o = sum_j P_j (s'_j c'_j + z'_j), codes c of 4 or 8 bits with a scale and a
// minimum a row.
//
// The pages are never expanded.  Codes enter the matrix products as what they
// are, small whole numbers, exact in bf16; the scale of a key multiplies its
// score behind the first product, that of a value its P before the second, and the
// minima add one number a head to the output.  So nothing of a key or value is
// rounded, and q enters as one, two or three bf16 terms (bf16, fp16, fp32: exact).
// P s' is the sum of two terms (fp32: three), of whose rounding 2^-17 (2^-25) is
// left.
//
// A code of 4 bits becomes a bf16 number by or-ing it into the mantissa of 16 (16
// + c is exact, and nothing is converted): two operations a pair of codes.  The 16
// is taken off again where the minima are added: -16 sum q starts the accumulator
// of the first product, and the second's share joins the minima's.  Codes of 8
// bits are converted through fp32.
//
// The blocks share the work as in nxa_paged.hip (units of 128 tokens, pieces of
// a row joined by its second kernel).  A step of a wave is 32 tokens, two halves
// of 16: S^T = K Q^T by 16x16x32 products a half, whose accumulator holds P^T as the
// second product reads it, O^T += V^T P^T over all 32.  Per half a lane loads a
// quarter of one key's codes (the head dim of a product is summed in any order,
// so q is read in the order of the codes), DP / 16 columns of four keys' values,
// and the scales of those four keys.
#include "nxa_quant.h"

#include "nxa_paged_units.h"

#include <type_traits>

namespace nxa {

namespace {

constexpr int kHalfKeys = 16;

template <typename T, int DP, int BITS>
struct QuantStep {
  static constexpr int ES = sizeof(T);
  static constexpr int NKW = DP * BITS / 128;      // dwords of K's codes a lane and half
  static constexpr int NJ = DP / 32;               // products of a half's S
  static constexpr int DPL = DP / 16;              // V columns of a lane
  static constexpr int VB = DPL * BITS / 8;        // bytes of them a key
  static constexpr int NVW = VB >= 4 ? VB / 4 : 1;  // dwords
  static constexpr int NS = ES;                    // dwords of a token's scales: 4 ES / 4
  static constexpr int QT = ES == 4 ? 3 : std::is_same<T, f16>::value ? 2 : 1;  // terms of q
  static constexpr int PT = ES == 4 ? 3 : 2;                                     // of P s'
};

template <typename T, int DP, int BITS>
struct HalfRegs {
  using R = QuantStep<T, DP, BITS>;
  Words<R::NKW> k;
  Words<R::NVW> v[4];
  Words<R::NS> s[4];
};

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two numbers as bf16, the first in the low half; and what their rounding left.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 r = {(bf16)a, (bf16)b};
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float low_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Whole bytes of a word as floats.
template <int B>
__device__ __forceinline__ float byte_of(uint32_t w) {
  return (float)(w >> (8 * B) & 255u);
}

// 16 + the nibbles at bits SH .. SH + 3 and SH + 16 .. SH + 19, as bf16: 16 is
// 0x4180, and a mantissa's unit is 2^-3 there.
template <int SH>
__device__ __forceinline__ uint32_t nibbles(uint32_t w) {
  const uint32_t x = SH < 3 ? w << (3 - SH) : w >> (SH - 3);
  return (x & 0x00780078u) | 0x41804180u;
}

// Product operand j of a lane's codes of one key: eight of them.
template <int BITS, int N>
__device__ __forceinline__ u32x4 key_operand(const Words<N>& k, int j) {
  if constexpr (BITS == 4) {
    const uint32_t w = k.w[j];
    return u32x4{nibbles<0>(w), nibbles<4>(w), nibbles<8>(w), nibbles<12>(w)};
  } else {
    const uint32_t a = k.w[2 * j], b = k.w[2 * j + 1];
    return u32x4{pack2(byte_of<0>(a), byte_of<1>(a)), pack2(byte_of<2>(a), byte_of<3>(a)),
                 pack2(byte_of<0>(b), byte_of<1>(b)), pack2(byte_of<2>(b), byte_of<3>(b))};
  }
}
// The element of the lane's eight that stands at place e of the operand.
template <int BITS>
__device__ constexpr int key_order(int e) {
  return BITS == 4 ? (e >> 1) + 4 * (e & 1) : e;
}

// Scales of a token: fields k's scale and minimum, v's.
template <typename T, int N>
__device__ __forceinline__ float scale_field(const Words<N>& s, int f) {
  if constexpr (std::is_same<T, float>::value) {
    return __uint_as_float(s.w[f]);
  } else if constexpr (std::is_same<T, f16>::value) {
    const uint16_t h = (uint16_t)(s.w[f >> 1] >> (16 * (f & 1)));
    return (float)__builtin_bit_cast(f16, h);
  } else {
    return f & 1 ? high_of(s.w[f >> 1]) : low_of(s.w[f >> 1]);
  }
}

}  // namespace

// Steps whose loads are in flight.
template <int DP, int BITS>
constexpr int kQuantDepth = DP * BITS <= 512 ? 3 : 2;

// FAST: pages hold a multiple of 16 tokens, so that a half lies in one page and
// its address is uniform, and no lane's codes straddle a row's end; else every key
// looks its page up and codes are loaded four bytes at a time.
template <typename T, int DP, int BITS, bool FAST>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void qpaged_kernel(const QuantPagedParams p) {
  using R = QuantStep<T, DP, BITS>;
  using Half = HalfRegs<T, DP, BITS>;
  constexpr int NKW = R::NKW, NJ = R::NJ, DPL = R::DPL, VB = R::VB, NVW = R::NVW, NS = R::NS;
  constexpr int QT = R::QT, PT = R::PT;
  constexpr int NB = kQuantDepth<DP, BITS>;
  constexpr int NF = DPL;  // O^T fragments: fragment f is columns DPL i + f, i = 0 .. 15
  constexpr int FIELDS = NF * 4 + 2;
  constexpr uint32_t kNowhere = 0x7ffffff0u;  // beyond every range
  __shared__ float ms[kWaves * FIELDS * 64];
  __shared__ int pre[257], wsum[kWaves];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int HV = p.Hk * p.strips;

  // The units of this block, u .. u1 (as in paged_kernel).
  int64_t u, u1, units = 0;
  int b, before, nblk = 0;
  if (p.nblk == 0) {
    b = blockIdx.x / HV;
    before = 0;
    const int n = paged_units(p, b), hv = blockIdx.x % HV;
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
    paged_prefix(p, pre, wsum);
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
    for (int n; before + (n = paged_units(p, b)) <= x; ++b) before += n;
    b = __builtin_amdgcn_readfirstlane(b);
    before = __builtin_amdgcn_readfirstlane(before);
  }
  const int64_t u0 = u;

  // Bytes of a row, and per-lane byte offsets inside a half: K key c, chunk g; V
  // key 4 g + j, columns DPL c ..; scales of key 4 g + j.
  const int kb = p.D * BITS / 8, vb = p.Dv * BITS / 8;
  uint32_t koff, voff[4];
  if constexpr (FAST) {
    koff = 4 * NKW * g < kb ? (uint32_t)(c * kb + 4 * NKW * g) : kNowhere;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      voff[j] = VB * c < vb ? (uint32_t)((4 * g + j) * vb + VB * c) : kNowhere;
  }

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

    // Q^T: column c is head h0 + c; the lane's quarter of the head dim in the
    // order of K's codes, as QT terms, and the sum of the whole row.
    u32x4 qf[NJ][QT];
    float qsum = 0.f;
    {
      const T* qp = (const T*)p.q + b * p.q_str[0] + ((int64_t)hk * p.G + h0 + min(c, heads - 1)) * p.q_str[1];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int d = g * (DP / 4) + 8 * j;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
        if (c < heads && d < p.D) {
          const u32x4* src = reinterpret_cast<const u32x4*>(qp + d);
          if constexpr (sizeof(T) == 4) {
            const f32x4 lo = __builtin_bit_cast(f32x4, src[0]), hi = __builtin_bit_cast(f32x4, src[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = lo[e], x[4 + e] = hi[e];
          } else {
            struct alignas(16) Row { T x[8]; };
            const Row y = __builtin_bit_cast(Row, src[0]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)y.x[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) qsum += x[e];
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float& a = x[key_order<BITS>(2 * w)];
            float& o = x[key_order<BITS>(2 * w + 1)];
            const uint32_t r = pack2(a, o);
            qf[j][t][w] = r;
            a -= low_of(r), o -= high_of(r);
          }
      }
      qsum += xor16(qsum);
      qsum += shfl_xor32(qsum);
    }
    const float qz = qsum * p.scale_log2;
    const float s_init = BITS == 4 ? -16.f * qsum : 0.f;
    f32x4 o[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (zs: what the minima, and 16 in the place of 0, add to every column)
    float m_ref = -INFINITY, l = 0.f, zs = 0.f;

    const char* kp = (const char*)p.k + hk * p.k_str[1];
    const char* vp = (const char*)p.v + hk * p.v_str[1];
    const T* sp = (const T*)p.sc + hk * p.sc_str[1];
    // This wave's steps: 32 tokens of each unit, up to the length.
    auto key_of = [&](int half) { return (t0 + (half >> 1)) * kPagedKeys + wave * 32 + (half & 1) * kHalfKeys; };
    int steps = t1 - t0;
    while (steps > 0 && key_of(2 * steps - 2) >= len) --steps;

    for (int i0 = 0; i0 < steps; i0 += 32) {
      const int ns = min(32, steps - i0);
      // Lane i looks up half 2 i0 + i: its page, its slot there and the tokens it
      // has (none where the table has no page).
      int page = 0, slot = 0, rows = 0;
      if (FAST && lane < 2 * ns) {
        const int key0 = key_of(2 * i0 + lane);
        if (key0 < len) {
          page = p.table[b * p.table_rs + key0 / p.PS];
          slot = key0 % p.PS;
          if ((unsigned)page < (unsigned)p.P) rows = min(kHalfKeys, len - key0);
          else page = 0;
        }
      }
      Half ring[NB][2];
      int have[NB][2];  // tokens of the half (FAST), or a bit a token
      auto issue = [&](int hi, Half& r, int& mine) NXA_INLINE {
        if constexpr (FAST) {
          // (past the last step: empty ranges, so every step counts alike)
          const int j = min(hi, 2 * ns - 1);
          const int nr = hi < 2 * ns ? __builtin_amdgcn_readlane(rows, j) : 0;
          const int64_t pg = __builtin_amdgcn_readlane(page, j);
          const int64_t sl = __builtin_amdgcn_readlane(slot, j);
          const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(kp + pg * p.k_str[0] + sl * kb), 0, nr * kb, 0x00020000);
          const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(vp + pg * p.v_str[0] + sl * vb), 0, nr * vb, 0x00020000);
          const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(sp + pg * p.sc_str[0] + sl * 4), 0, nr * 4 * R::ES, 0x00020000);
          r.k = buf_load<NKW>(rk, koff);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if constexpr (VB == 2)
              r.v[x].w[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rv, voff[x], 0, kNonTemporal);
            else
              r.v[x] = buf_load<NVW>(rv, voff[x]);
          }
          // (a load a token, so that none straddles the range's end)
#pragma unroll
          for (int x = 0; x < 4; ++x) r.s[x] = buf_load<NS>(rs, (4 * g + x) * 4 * R::ES);
          mine = nr;
        } else {
          // Lane x < 16 looks up token x of the half; the others ask it.
          const int key = key_of(2 * i0 + min(hi, 2 * ns - 1)) + c;
          int pg = -1, sl = 0;
          if (hi < 2 * ns && key < len) {
            pg = p.table[b * p.table_rs + key / p.PS];
            sl = key % p.PS;
          }
          const bool ok = (unsigned)pg < (unsigned)p.P;
          if (!ok) pg = sl = 0;
          mine = (int)(__ballot(ok) & 0xffff);
          const char* kr = kp + pg * p.k_str[0] + (int64_t)sl * kb + 4 * NKW * g;
#pragma unroll
          for (int w = 0; w < NKW; ++w)
            r.k.w[w] = ok && 4 * (NKW * g + w) < kb ? reinterpret_cast<const uint32_t*>(kr)[w] : 0u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int src = 4 * g + x;
            const bool on = mine >> src & 1;
            const int64_t vpg = __shfl(pg, src, 64), vsl = __shfl(sl, src, 64);
            const char* vr = vp + vpg * p.v_str[0] + vsl * vb + VB * c;
            if constexpr (VB == 2) {
              r.v[x].w[0] = on && VB * c < vb ? *reinterpret_cast<const uint16_t*>(vr) : 0u;
            } else {
#pragma unroll
              for (int w = 0; w < NVW; ++w)
                r.v[x].w[w] = on && VB * c + 4 * w < vb ? reinterpret_cast<const uint32_t*>(vr)[w] : 0u;
            }
            const uint32_t* sr = reinterpret_cast<const uint32_t*>(sp + vpg * p.sc_str[0] + vsl * 4);
#pragma unroll
            for (int w = 0; w < NS; ++w) r.s[x].w[w] = on ? sr[w] : 0u;
          }
        }
      };
      auto compute = [&](const Half (&r)[2], const int (&mine)[2]) NXA_INLINE {
        f32x4 s[2];
        float mt = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s[h] = f32x4{s_init, s_init, s_init, s_init};
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const u32x4 a = key_operand<BITS>(r[h].k, j);
#pragma unroll
            for (int t = 0; t < QT; ++t) s[h] = mma(a, qf[j][t], s[h]);
          }
          // Rows of the accumulator: tokens 4 g + e.
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool ok = FAST ? 4 * g + e < mine[h] : (mine[h] >> (4 * g + e) & 1) != 0;
            // (a scale of infinity makes its token NaN, whatever the signs)
            const float ks = scale_field<T>(r[h].s[e], 0), kz = scale_field<T>(r[h].s[e], 1);
            const float x = __builtin_fmaf(s[h][e], ks * p.scale_log2, __builtin_fmaf(kz, qz, ks * 0.f));
            s[h][e] = ok ? x : -INFINITY;
            mt = fmaxf(mt, s[h][e]);
          }
        }
        if (__any(mt > m_ref + kSlack)) {
          mt = fmaxf(mt, xor16(mt));
          mt = fmaxf(mt, shfl_xor32(mt));
          const float mn = fmaxf(m_ref, mt);
          const float alpha = mn > m_ref ? fast_exp2(m_ref - mn) : 1.f;
          l *= alpha;
          zs *= alpha;
#pragma unroll
          for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[f][e] *= alpha;
          m_ref = mn;
        }
        const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
        float x[8];  // P s'
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = fast_exp2(s[h][e] + neg_m);
            const float sc = scale_field<T>(r[h].s[e], 2), z = scale_field<T>(r[h].s[e], 3);
            l += w;
            x[4 * h + e] = w * sc;
            zs = __builtin_fmaf(w, BITS == 4 ? __builtin_fmaf(-16.f, sc, z) : z, zs);
          }
        u32x4 pf[PT];
#pragma unroll
        for (int t = 0; t < PT; ++t)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            pf[t][w] = pack2(x[2 * w], x[2 * w + 1]);
            x[2 * w] -= low_of(pf[t][w]);
            x[2 * w + 1] -= high_of(pf[t][w]);
          }
        auto product = [&](int f, u32x4 a) NXA_INLINE {
#pragma unroll
          for (int t = 0; t < PT; ++t) o[f] = mma(a, pf[t], o[f]);
        };
#pragma unroll
        for (int w = 0; w < NVW; ++w)
#pragma unroll
          for (int y = 0; y < (VB < 4 ? VB : 4); ++y) {
            // Byte y of word w of the lane's eight keys, in pairs.
            const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + y) << 16 | (uint32_t)y;
            uint32_t t[4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                t[2 * h + e] = __builtin_amdgcn_perm(r[h].v[2 * e + 1].w[w], r[h].v[2 * e].w[w], sel);
            if constexpr (BITS == 4) {
              product(8 * w + 2 * y, u32x4{nibbles<0>(t[0]), nibbles<0>(t[1]), nibbles<0>(t[2]), nibbles<0>(t[3])});
              product(8 * w + 2 * y + 1, u32x4{nibbles<4>(t[0]), nibbles<4>(t[1]), nibbles<4>(t[2]), nibbles<4>(t[3])});
            } else {
              u32x4 a;
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] = pack2(byte_of<0>(t[e]), byte_of<2>(t[e]));
              product(4 * w + y, a);
            }
          }
      };
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) issue(2 * x + h, ring[x][h], have[x][h]);
      for (int i = 0; i < ns; i += NB)
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          compute(ring[x], have[x]);
#pragma unroll
          for (int h = 0; h < 2; ++h) issue(2 * (i + x + NB) + h, ring[x][h], have[x][h]);
        }
    }
    l += xor16(l);
    l += shfl_xor32(l);
    zs += xor16(zs);
    zs += shfl_xor32(zs);

    // Join the waves: [wave][field][lane], field 4 f + e of O, then m and l.
    __syncthreads();
    {
      float* mw = ms + wave * FIELDS * 64 + lane;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) mw[(4 * f + e) * 64] = o[f][e] + zs;
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
    u += v1 - v0;
    if (hv == HV - 1 && v1 == n) {
      before += n;
      ++b;
    }
  }
}

int qpaged_dp(int m) { return m <= 64 ? 64 : m <= 128 ? 128 : 256; }

bool qpaged_whole(int64_t room) { return room <= 1024; }

template <typename T, int DP, int BITS>
static void launch_qpaged_b(const QuantPagedParams& p, hipStream_t stream) {
  const dim3 grid(p.nblk ? p.nblk : p.B * p.Hk * p.strips), block(256);
  using R = QuantStep<T, DP, BITS>;
  const int kb = p.D * BITS / 8, vb = p.Dv * BITS / 8;
  if (p.PS % kHalfKeys == 0 && kb % (4 * R::NKW) == 0 && vb % R::VB == 0)
    hipLaunchKernelGGL((qpaged_kernel<T, DP, BITS, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((qpaged_kernel<T, DP, BITS, false>), grid, block, 0, stream, p);
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
