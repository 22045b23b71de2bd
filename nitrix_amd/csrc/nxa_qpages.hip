// New tokens into quantised pages and back (nxa_quant.h).
//
// A block takes kTokens tokens: a thread each finds a token's sequence and page, and
// then a wave takes one, LPR lanes of eight elements a row (a head's key or value),
// 64 / LPR rows at a time.  A row is read (written) once in the model's type and
// written (read) once in codes.  Reading back is bound by HBM: 65,664 tokens of 8 heads
// of 128 in bf16 and 4 bits 56 us, 6.1 TB/s, 16384 tokens 17 us.  Writing 16384 takes 28
// us (3.1 TB/s): some 170 vector operations for a lane's eight elements, which keep
// the SIMDs busy for three quarters of it.  What hides latency is waves, eight a SIMD: with
// two or four such steps loaded together a wave held 99 or more registers in place of 53,
// and writing took 39 and 47 us, 31 then; 16 tokens a block took 35, and 1024 tokens in 8
// bits 13 in place of 9.
//
// Codes are rounded as the exact quotient would be, ties to even, so that they do
// not depend on how it is taken (exact_code; near_code where it is as good).
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

// Past the caches: 65,664 tokens of 8 heads of 128 read back in 56 us in place of 95.
template <typename T>
__device__ __forceinline__ void store_eight(T* at, const Eight<T>& y) {
  const u32x4* src = reinterpret_cast<const u32x4*>(&y);
  u32x4* dst = reinterpret_cast<u32x4*>(at);
#pragma unroll
  for (int i = 0; i < (int)sizeof(y) / 16; ++i) __builtin_nontemporal_store(src[i], dst + i);
}

constexpr int kTokens = 4;  // of a block, a wave each

// Where the tokens of a block are: a page (none: -1) and a slot.  Threads 0 ..
// kTokens - 1, a token each; `ends` (LDS) holds the offsets where these are few.
constexpr int kFewOffsets = 1024;
struct Place {
  int page, slot;
};
__device__ __forceinline__ Place quant_place(const QuantMoveParams& p, int64_t t, const int* ends) {
  Place at = {-1, 0};
  if (t >= p.T) return at;
  int64_t s = t, pos = 0;
  if (p.offsets) {
    const bool few = p.B < kFewOffsets;
    int lo = 0, hi = p.B + 1;  // last s with offsets[s] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((few ? ends[mid] : p.offsets[mid]) <= t) lo = mid;
      else hi = mid;
    }
    const int start = few ? ends[lo] : p.offsets[lo];
    if (lo >= p.B || start > t) return at;
    s = lo;
    pos = t - start;
  }
  pos += p.starts[s];
  if (pos < 0 || pos >= (int64_t)p.M * p.pool.PS) return at;
  const int page = p.table[s * p.table_rs + pos / p.pool.PS];
  if ((unsigned)page >= (unsigned)p.pool.P) return at;
  at.page = page;
  at.slot = (int)(pos % p.pool.PS);
  return at;
}
__device__ __forceinline__ void quant_places(const QuantMoveParams& p, int64_t t0, Place* place) {
  __shared__ int ends[kFewOffsets];
  if (p.offsets && p.B < kFewOffsets) {
    for (int i = threadIdx.x; i <= p.B; i += 64 * kTokens) ends[i] = p.offsets[i];
    __syncthreads();
  }
  if (threadIdx.x < kTokens) place[threadIdx.x] = quant_place(p, t0 + threadIdx.x, ends);
  __syncthreads();
}

// Reductions over the LPR lanes of a row; every lane has the result.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
template <int LPR, typename F>
__device__ __forceinline__ uint32_t row_reduce(uint32_t x, F&& f) {
  x = f(x, dpp<0xb1>(x));   // lanes 1, 0, 3, 2 of each four
  x = f(x, dpp<0x4e>(x));   // 2, 3, 0, 1
  x = f(x, dpp<0x141>(x));  // each eight mirrored
  if constexpr (LPR >= 16) x = f(x, dpp<0x140>(x));  // each sixteen
  if constexpr (LPR >= 32) x = f(x, (uint32_t)__shfl_xor((int)x, 16, 64));
  return x;
}
// (NaN where one of them is)
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("v_minimum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
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

// The same where x - z is exact in fp32 and s has few bits (16-bit types, x and z
// not too far apart): the quotient by the reciprocal, corrected by its remainder, is
// the exact one but for 2^-45 of it, rounded to fp32 (inv is off by a place or two).
// A border n + 1/2 is an fp32 number, and (n + 1/2) s, of 20 bits or fewer, stands in
// the places of x - z: one that is not a border differs from it by a place of x - z or
// more, at least 1 + 2^-11 times half a place of the quotient (s has 11 bits or fewer),
// and is not rounded to it.
__device__ __forceinline__ float near_code(float diff, float s, float inv) {
  const float q = diff * inv;
  return __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, s, diff), inv, q));
}

}  // namespace

// Eight elements of a row of keys or values into codes at dst, by LPR lanes (those
// behind the row's end not `mine`); the row's scale and minimum at sc.
template <typename T, int BITS, int LPR>
__device__ __forceinline__ void write_row(const Eight<T>& y, bool mine, bool first, char* dst,
                                          T* sc) {
  constexpr int TOP = (1 << BITS) - 1;
  // x - z is exact where neither is 2^FAR times the other or more: 24 places less
  // the 8 of bf16 or the 11 of fp16.
  constexpr int FAR = std::is_same<T, f16>::value ? 12 : 15;
  constexpr float kFar = 1 << FAR;
  float x[8], lo = INFINITY, hi = -INFINITY;
  uint32_t least = 0xffffffffu;  // twice the bits of the least |x| but 0, less one
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)y.x[e];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    lo = min3(lo, x[e], x[e + 1]);
    hi = max3(hi, x[e], x[e + 1]);
    least = min(least, min(2u * __float_as_uint(x[e]) - 1u, 2u * __float_as_uint(x[e + 1]) - 1u));
  }
  const float far = fmaxf(__builtin_fabsf(lo), __builtin_fabsf(hi));
  if (!mine) lo = INFINITY, hi = -INFINITY;
  lo = __uint_as_float(row_reduce<LPR>(__float_as_uint(lo), [](uint32_t a, uint32_t b) {
    return __float_as_uint(min3(__uint_as_float(a), __uint_as_float(b), INFINITY));
  }));
  hi = __uint_as_float(row_reduce<LPR>(__float_as_uint(hi), [](uint32_t a, uint32_t b) {
    return __float_as_uint(max3(__uint_as_float(a), __uint_as_float(b), -INFINITY));
  }));
  // (a row of NaN, infinity or a range past fp32's reads back as NaN)
  const float range = hi - lo;
  const bool bad = !(range < INFINITY);
  const T zt = (T)(bad ? NAN : lo), st = (T)(bad ? NAN : range * (1.f / TOP));
  const float z = (float)zt;
  float sf = (float)st;
  // (quotients of tiny scales are taken 2^96 times larger)
  const float up = sf < 0x1p-90f ? 0x1p96f : 1.f;
  sf *= up;
  // (the hardware's reciprocal, off by a place or so, and a step that leaves next to
  // nothing of that)
  const float near_inv = __builtin_amdgcn_rcpf(sf);
  const float inv =
      sf > 0.f ? __builtin_fmaf(__builtin_fmaf(-sf, near_inv, 1.f), near_inv, near_inv) : 0.f;
  float n[8];
  const float az = __builtin_fabsf(z);
  const bool near = sizeof(T) == 2 && up == 1.f &&
                    __uint_as_float((least + 1u) >> 1) >= az * (1.f / kFar) &&
                    (far <= az * kFar || z == 0.f);
  if (__builtin_expect(__any(!near && mine), 0)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = exact_code(x[e] * up, z * up, sf, inv);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = near_code(x[e] - z, sf, inv);
  }
  // (a scale of zero or NaN gives 0, what is below the stored minimum too)
#pragma unroll
  for (int e = 0; e < 8; ++e) n[e] = fminf(fmaxf(n[e], 0.f), (float)TOP);
  if (!mine) return;
  // Codes put together as whole numbers that fp32 holds: four of 4 bits, two of 8.
  auto pair = [&](int e) { return __builtin_fmaf(n[e + 1], (float)(TOP + 1), n[e]); };
  if constexpr (BITS == 4) {
    const float a = __builtin_fmaf(pair(2), 256.f, pair(0)), b = __builtin_fmaf(pair(6), 256.f, pair(4));
    *reinterpret_cast<uint32_t*>(dst) = (uint32_t)a | (uint32_t)b << 16;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<uint32_t*>(dst)[i] =
          (uint32_t)pair(4 * i) | (uint32_t)pair(4 * i + 2) << 16;
  }
  if (first) {
    struct alignas(2 * sizeof(T)) Scale {
      T s, z;
    };
    *reinterpret_cast<Scale*>(sc) = {st, zt};
  }
}

template <typename T, int BITS, int LPR>
__global__ __launch_bounds__(64 * kTokens) void quant_write_kernel(const QuantMoveParams p) {
  constexpr int RG = 64 / LPR;
  __shared__ Place place[kTokens];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t = (int64_t)blockIdx.x * kTokens + wave;
  const QuantPool& pool = p.pool;
  const int sub = lane % LPR, d = 8 * sub, h1 = lane / LPR;
  const bool in_k = d < pool.D, in_v = d < pool.Dv;
  const T* ks = (const T*)p.ks + h1 * p.ks_str[0] + d;
  const T* vs = (const T*)p.vs + h1 * p.vs_str[0] + d;
  char* kd = (char*)pool.k + h1 * pool.k_str[1] + d * BITS / 8;
  char* vd = (char*)pool.v + h1 * pool.v_str[1] + d * BITS / 8;
  T* sd = (T*)pool.sc + h1 * pool.sc_str[1];
  quant_places(p, t - wave, place);
  if (t >= p.T) return;
  const int page = __builtin_amdgcn_readfirstlane(place[wave].page);
  const int slot = __builtin_amdgcn_readfirstlane(place[wave].slot);
  if (page < 0) return;
  const int64_t ko = page * pool.k_str[0] + (int64_t)slot * (pool.D * BITS / 8);
  const int64_t vo = page * pool.v_str[0] + (int64_t)slot * (pool.Dv * BITS / 8);
  const int64_t so = page * pool.sc_str[0] + 4 * (int64_t)slot;
  const int64_t kt = t * p.ks_str[1], vt = t * p.vs_str[1];
  for (int h = 0; h + h1 < pool.Hk; h += RG) {  // (this lane's head is h + h1)
    Eight<T> k = {}, v = {};
    if (in_k) k = load_eight(ks + kt + h * p.ks_str[0]);
    if (in_v) v = load_eight(vs + vt + h * p.vs_str[0]);
    T* sc = sd + so + h * pool.sc_str[1];
    write_row<T, BITS, LPR>(k, in_k, sub == 0, kd + ko + h * pool.k_str[1], sc);
    write_row<T, BITS, LPR>(v, in_v, sub == 0, vd + vo + h * pool.v_str[1], sc + 2);
  }
}

// A lane's eight codes and its row's scale and minimum.
template <typename T, int BITS>
struct HeldRow {
  uint32_t w[BITS / 4];
  struct alignas(2 * sizeof(T)) Scale {
    T s, z;
  } sc;
  __device__ __forceinline__ void load(const char* src, const T* at) {
#pragma unroll
    for (int x = 0; x < BITS / 4; ++x) w[x] = reinterpret_cast<const uint32_t*>(src)[x];
    sc = *reinterpret_cast<const Scale*>(at);
  }
  __device__ __forceinline__ Eight<T> values() const {
    const float a = (float)sc.s, z = (float)sc.z;
    // (a scale is rounded, up too, so that the largest code of a row that ends near the
    // type's largest number may stand for more than that)
    constexpr float MOST = std::is_same<T, f16>::value ? 65504.f : sizeof(T) == 2 ? 0x1.fep127f : 0x1.fffffep127f;
    const float lim = a < INFINITY && z < INFINITY ? MOST : INFINITY;
    Eight<T> y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = BITS == 4 ? w[0] >> (4 * e) & 15 : w[e / 4 % (BITS / 4)] >> (8 * (e % 4)) & 255;
      y.x[e] = (T)min3(__builtin_fmaf((float)c, a, z), lim, lim);
    }
    return y;
  }
};

template <typename T, int BITS, int LPR>
__global__ __launch_bounds__(64 * kTokens) void quant_read_kernel(const QuantMoveParams p) {
  constexpr int RG = 64 / LPR;
  __shared__ Place place[kTokens];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t = (int64_t)blockIdx.x * kTokens + wave;
  const QuantPool& pool = p.pool;
  const int sub = lane % LPR, d = 8 * sub, h1 = lane / LPR;
  const bool in_k = d < pool.D, in_v = d < pool.Dv;
  T* kd = (T*)p.ks + h1 * p.ks_str[0] + d;
  T* vd = (T*)p.vs + h1 * p.vs_str[0] + d;
  const char* ks = (const char*)pool.k + h1 * pool.k_str[1] + d * BITS / 8;
  const char* vs = (const char*)pool.v + h1 * pool.v_str[1] + d * BITS / 8;
  const T* ss = (const T*)pool.sc + h1 * pool.sc_str[1];
  quant_places(p, t - wave, place);
  if (t >= p.T) return;
  const int page = __builtin_amdgcn_readfirstlane(place[wave].page);
  const int slot = __builtin_amdgcn_readfirstlane(place[wave].slot);
  const int64_t ko = page * pool.k_str[0] + (int64_t)slot * (pool.D * BITS / 8);
  const int64_t vo = page * pool.v_str[0] + (int64_t)slot * (pool.Dv * BITS / 8);
  const int64_t so = page * pool.sc_str[0] + 4 * (int64_t)slot;
  const int64_t kt = t * p.ks_str[1], vt = t * p.vs_str[1];
  for (int h = 0; h + h1 < pool.Hk; h += RG) {  // (this lane's head is h + h1)
    HeldRow<T, BITS> k = {}, v = {};            // (zero where there is no page)
    if (page >= 0) {
      const T* at = ss + so + h * pool.sc_str[1];
      if (in_k) k.load(ks + ko + h * pool.k_str[1], at);
      if (in_v) v.load(vs + vo + h * pool.v_str[1], at + 2);
    }
    if (in_k) store_eight(kd + kt + h * p.ks_str[0], k.values());
    if (in_v) store_eight(vd + vt + h * p.vs_str[0], v.values());
  }
}

template <typename T, int BITS, bool WRITE>
static void launch_move_t(const QuantMoveParams& p, hipStream_t stream) {
  const int most = p.pool.D > p.pool.Dv ? p.pool.D : p.pool.Dv;
  auto go = [&](auto lpr) {
    constexpr int LPR = decltype(lpr)::value;
    const dim3 grid((unsigned)((p.T + kTokens - 1) / kTokens)), block(64 * kTokens);
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
