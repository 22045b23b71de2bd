// New tokens into quantised pages and back (nxa_quant.h).
//
// A wave a token: it finds the token's sequence and page once and then takes the
// rows of all heads, keys and values, LPR lanes of eight elements a row and 64 /
// LPR rows at a time.  Bound by HBM: a row is read (written) once in the model's
// type and written (read) once in codes.
//
// Codes are rounded as the exact quotient would be, ties to even, so that they do
// not depend on how it is taken (exact_code).
#include "nxa_quant.h"

#include <type_traits>

namespace nxa {

namespace {

// Eight consecutive elements of a lane.
template <typename T>
struct alignas(16) Eight {
  T x[8];
};

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* at) {
  Eight<T> r;
  const u32x4* src = reinterpret_cast<const u32x4*>(at);
  u32x4* dst = reinterpret_cast<u32x4*>(&r);
#pragma unroll
  for (int i = 0; i < (int)sizeof(r) / 16; ++i) dst[i] = __builtin_nontemporal_load(src + i);
  return r;
}

// Sequence and position of token t (whole wave; uniform); false: of no sequence
// or outside the table.
__device__ __forceinline__ bool quant_find(const QuantMoveParams& p, int64_t t, int& s,
                                           int64_t& pos) {
  const int lane = threadIdx.x & 63;
  s = (int)t;
  pos = 0;
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
    if (s >= p.B || p.offsets[s] > t) return false;
    pos = t - p.offsets[s];
  }
  pos += p.starts[s];
  return pos >= 0 && pos < (int64_t)p.M * p.pool.PS;
}

// rint((x - z) / s) of the exact quotient, given s and (roughly) 1 / s; zero
// where s is zero or NaN.  The quotient by the reciprocal is off by less than a
// step; what is left of x - z then settles it: x - z is the sum of two numbers,
// the second what the first rounded off, and a fused multiply-add takes n s from
// the first exactly (both are whole multiples of the last place of s or of half of
// it, and little more than s / 2 is left).
__device__ __forceinline__ float exact_code(float x, float z, float s, float inv) {
  const float diff = x - z, part = diff - x;
  const float low = (x - (diff - part)) - (z + part);
  float n = __builtin_rintf(diff * inv);
  const float rest = __builtin_fmaf(-n, s, diff), half = 0.5f * s;
  const float over = (rest - half) + low, under = (rest + half) + low;
  const bool odd = (int)n & 1;
  if (over > 0.f || (over == 0.f && odd)) n += 1.f;
  else if (under < 0.f || (under == 0.f && odd)) n -= 1.f;
  return s > 0.f ? n : 0.f;
}

}  // namespace

template <typename T, int BITS, int LPR>
__global__ __launch_bounds__(256) void quant_write_kernel(const QuantMoveParams p) {
  constexpr int TOP = (1 << BITS) - 1;
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.T) return;
  int s;
  int64_t pos;
  if (!quant_find(p, t, s, pos)) return;
  const QuantPool& pool = p.pool;
  const int page = p.table[s * p.table_rs + pos / pool.PS];
  if ((unsigned)page >= (unsigned)pool.P) return;
  const int slot = (int)(pos % pool.PS);
  const int sub = lane % LPR, d = 8 * sub;
  for (int r = lane / LPR; r < 2 * pool.Hk; r += 64 / LPR) {
    const int which = r >= pool.Hk, h = which ? r - pool.Hk : r;
    const int D = which ? pool.Dv : pool.D;
    const T* src = which ? (const T*)p.vs + h * p.vs_str[0] + t * p.vs_str[1]
                         : (const T*)p.ks + h * p.ks_str[0] + t * p.ks_str[1];
    float x[8], lo = INFINITY, hi = -INFINITY, bad = 0.f;
    if (d < D) {
      const Eight<T> y = load_eight(src + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = (float)y.x[e];
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
        bad = __builtin_fmaf(x[e], 0.f, bad);  // NaN where x is NaN or infinite
      }
    }
#pragma unroll
    for (int m = 1; m < LPR; m *= 2) {
      lo = fminf(lo, __shfl_xor(lo, m, 64));
      hi = fmaxf(hi, __shfl_xor(hi, m, 64));
      bad += __shfl_xor(bad, m, 64);
    }
    // (a row of NaN, infinity or a range past the type's reads back as NaN)
    const float range = hi - lo;
    bad = __builtin_fmaf(range, 0.f, bad);
    const T zt = (T)(lo + bad), st = (T)(range * (1.f / TOP) + bad);
    const float z = (float)zt;
    float sf = (float)st;
    // (quotients of tiny scales are taken 2^96 times larger)
    const float up = sf < 0x1p-90f ? 0x1p96f : 1.f;
    sf *= up;
    const float inv = sf > 0.f ? 1.f / sf : 0.f;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = (uint32_t)fminf(fmaxf(exact_code(x[e] * up, z * up, sf, inv), 0.f), (float)TOP);
    if (d < D) {
      char* dst = which ? (char*)pool.v + page * pool.v_str[0] + h * pool.v_str[1]
                        : (char*)pool.k + page * pool.k_str[0] + h * pool.k_str[1];
      dst += (int64_t)slot * (D * BITS / 8) + d * BITS / 8;
      if constexpr (BITS == 4) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= c[e] << (4 * e);
        *reinterpret_cast<uint32_t*>(dst) = w;
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e / 4] |= c[e] << (8 * (e % 4));
        *reinterpret_cast<uint32_t*>(dst) = w[0];
        *reinterpret_cast<uint32_t*>(dst + 4) = w[1];
      }
      if (sub == 0) {
        T* sc = (T*)pool.sc + page * pool.sc_str[0] + h * pool.sc_str[1] + 4 * (int64_t)slot;
        sc[2 * which] = st;
        sc[2 * which + 1] = zt;
      }
    }
  }
}

template <typename T, int BITS, int LPR>
__global__ __launch_bounds__(256) void quant_read_kernel(const QuantMoveParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.T) return;
  const QuantPool& pool = p.pool;
  int s, page = -1, slot = 0;
  int64_t pos;
  if (quant_find(p, t, s, pos)) {
    page = p.table[s * p.table_rs + pos / pool.PS];
    slot = (int)(pos % pool.PS);
  }
  const bool held = (unsigned)page < (unsigned)pool.P;
  const int sub = lane % LPR, d = 8 * sub;
  for (int r = lane / LPR; r < 2 * pool.Hk; r += 64 / LPR) {
    const int which = r >= pool.Hk, h = which ? r - pool.Hk : r;
    const int D = which ? pool.Dv : pool.D;
    if (d >= D) continue;
    Eight<T> y;
    if (held) {
      const char* src = which ? (const char*)pool.v + page * pool.v_str[0] + h * pool.v_str[1]
                              : (const char*)pool.k + page * pool.k_str[0] + h * pool.k_str[1];
      src += (int64_t)slot * (D * BITS / 8) + d * BITS / 8;
      const T* sc =
          (const T*)pool.sc + page * pool.sc_str[0] + h * pool.sc_str[1] + 4 * (int64_t)slot;
      const float a = (float)sc[2 * which], z = (float)sc[2 * which + 1];
      const uint32_t w0 = *reinterpret_cast<const uint32_t*>(src);
      const uint32_t w1 = BITS == 8 ? *reinterpret_cast<const uint32_t*>(src + 4) : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = BITS == 4 ? w0 >> (4 * e) & 15 : (e < 4 ? w0 : w1) >> (8 * (e % 4)) & 255;
        y.x[e] = (T)__builtin_fmaf((float)c, a, z);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y.x[e] = (T)0.f;
    }
    T* dst = which ? (T*)p.vs + h * p.vs_str[0] + t * p.vs_str[1]
                   : (T*)p.ks + h * p.ks_str[0] + t * p.ks_str[1];
    *reinterpret_cast<Eight<T>*>(dst + d) = y;
  }
}

template <typename T, int BITS, bool WRITE>
static void launch_move_t(const QuantMoveParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.T + 3) / 4)), block(256);
  const int most = p.pool.D > p.pool.Dv ? p.pool.D : p.pool.Dv;
  auto go = [&](auto lpr) {
    constexpr int LPR = decltype(lpr)::value;
    if constexpr (WRITE)
      hipLaunchKernelGGL((quant_write_kernel<T, BITS, LPR>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((quant_read_kernel<T, BITS, LPR>), grid, block, 0, stream, p);
  };
  if (most <= 64) go(std::integral_constant<int, 8>());
  else if (most <= 128) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 32>());
}

template <bool WRITE>
static void launch_move(const QuantMoveParams& p, int io_dtype, hipStream_t stream) {
  const bool four = p.pool.bits == 4;
  if (io_dtype == kF32) {
    if (four) launch_move_t<float, 4, WRITE>(p, stream);
    else launch_move_t<float, 8, WRITE>(p, stream);
  } else if (io_dtype == kF16) {
    if (four) launch_move_t<f16, 4, WRITE>(p, stream);
    else launch_move_t<f16, 8, WRITE>(p, stream);
  } else {
    if (four) launch_move_t<bf16, 4, WRITE>(p, stream);
    else launch_move_t<bf16, 8, WRITE>(p, stream);
  }
}

void launch_quant_write(const QuantMoveParams& p, int io_dtype, hipStream_t stream) {
  launch_move<true>(p, io_dtype, stream);
}
void launch_quant_read(const QuantMoveParams& p, int io_dtype, hipStream_t stream) {
  launch_move<false>(p, io_dtype, stream);
}

}  // namespace nxa
