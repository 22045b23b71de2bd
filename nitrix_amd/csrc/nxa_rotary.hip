// Rotary positions: pairs of a row's elements turned by an angle that grows
// with the row's position,
//   a' = c (a cos pw - b sin pw),   b' = c (b cos pw + a sin pw),
// pair i of the half layout being elements i and i + R / 2, of the interleaved
// one 2 i and 2 i + 1; elements from R on are copied.  The backward pass is the
// same with the sines' sign turned.
//
// Bound by HBM: 6 operations on 4 bytes read and 4 written (16 bits).  What
// could cost more is the sine and cosine of each pair, which all heads of a
// token share: a block takes a token or a few with all their heads, forms each
// pair's once and keeps them in LDS.  Angles are turns, p w / (2 pi) with what the two
// products in 64 bits round off, of which the fraction goes on in 32 bits: positions
// up to 2^53 cost no accuracy (p (w / 2 pi) alone would be off by 2^-53 of itself).
// 16384 tokens of 40 heads of 128 in bf16 take 61 us (5.5 TB/s).
#include "nxa_rotary.h"

#include <type_traits>

namespace nxa {

namespace {

__device__ __forceinline__ int64_t rotary_position(const RotaryParams& p, int b, int t) {
  const int64_t at = b * p.pos_str[0] + t * p.pos_str[1];
  return p.pos64 ? ((const int64_t*)p.positions)[at] : ((const int*)p.positions)[at];
}

// c cos and c sin of pair i at a position.
__device__ __forceinline__ float2 rotary_turn(const RotaryParams& p, int64_t pos, int i) {
  // (1 / (2 pi) in two numbers)
  constexpr double kInvTwoPi = 0x1.45f306dc9c883p-3, kInvRest = -0x1.6b01ec5417056p-57;
  const double w = p.freq[i], a = (double)pos * w, a_rest = __builtin_fma((double)pos, w, -a);
  const double whole = __builtin_rint(a * kInvTwoPi);
  const double rest = __builtin_fma(a, kInvRest, a_rest * kInvTwoPi);
  const float f = (float)(2.0 * (__builtin_fma(a, kInvTwoPi, -whole) + rest));
  float s, c;
  sincospif(f, &s, &c);
  return float2{c * p.scale, (p.inverse ? -s : s) * p.scale};
}

template <typename T>
struct alignas(16) Chunk {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};

// Sixteen bytes to memory, of many tokens past the caches: us called in turn with /
// without, 8192 tokens of 40 heads of 128 in fp16 28.6 / 35.0, 16384 in bf16 53 / 66.
template <int TB, typename C>
__device__ __forceinline__ void put(void* at, const C& x) {
  u32x4* to = reinterpret_cast<u32x4*>(at);
  if (TB > 1) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x), to);
  else *to = __builtin_bit_cast(u32x4, x);
}

}  // namespace

// Rows as 16-byte chunks: an item is a pair of chunks that turn together (half
// layout), one chunk of pairs (interleaved) or one that is copied.  TB tokens a
// block.
template <typename T, bool IL, int TB>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  constexpr int N = Chunk<T>::N;
  __shared__ float2 cs[TB * kRotaryMaxDim / 2];
  const int tid = threadIdx.x, half = p.R / 2;
  const int blocks = (p.T + TB - 1) / TB;
  const int b = blockIdx.x / blocks, t0 = (blockIdx.x % blocks) * TB;
  const int nt = min(TB, p.T - t0);
  for (int i = tid; i < nt * half; i += 256) {
    const int t = i / half, j = i - t * half;
    cs[t * (kRotaryMaxDim / 2) + j] = rotary_turn(p, rotary_position(p, b, t0 + t), j);
  }
  __syncthreads();
  const int turned = IL ? p.R / N : half / N;
  const int per = turned + (p.D - p.R) / N, heads = p.H[0] + p.H[1];
  const int total = nt * heads * per;
  for (int i = tid; i < total; i += 256) {
    const int row = i / per, c = i - row * per;
    const int t = row / heads, hh = row - t * heads;
    const int w = hh >= p.H[0], h = w ? hh - p.H[0] : hh;
    const T* x = (const T*)p.x[w] + b * p.x_str[w][0] + h * p.x_str[w][1] + (t0 + t) * p.x_str[w][2];
    T* y = (T*)p.y[w] + b * p.y_str[w][0] + h * p.y_str[w][1] + (t0 + t) * p.y_str[w][2];
    const float2* at = cs + t * (kRotaryMaxDim / 2);
    if (c >= turned) {
      const int d = p.R + (c - turned) * N;
      put<TB>(y + d, *reinterpret_cast<const u32x4*>(x + d));
    } else if (IL) {
      Chunk<T> a = *reinterpret_cast<const Chunk<T>*>(x + c * N);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        const float2 k = at[c * (N / 2) + e];
        const float u = (float)a.x[2 * e], v = (float)a.x[2 * e + 1];
        a.x[2 * e] = (T)(u * k.x - v * k.y);
        a.x[2 * e + 1] = (T)(v * k.x + u * k.y);
      }
      put<TB>(y + c * N, a);
    } else {
      Chunk<T> a = *reinterpret_cast<const Chunk<T>*>(x + c * N);
      Chunk<T> o = *reinterpret_cast<const Chunk<T>*>(x + half + c * N);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 k = at[c * N + e];
        const float u = (float)a.x[e], v = (float)o.x[e];
        a.x[e] = (T)(u * k.x - v * k.y);
        o.x[e] = (T)(v * k.x + u * k.y);
      }
      put<TB>(y + c * N, a);
      put<TB>(y + half + c * N, o);
    }
  }
}

// Any head dim, rotated part, strides and alignment: a pair or an element an
// item (173 us where chunks take 61).
template <typename T, int TB>
__global__ __launch_bounds__(256) void rotary_any_kernel(const RotaryParams p) {
  __shared__ float2 cs[TB * kRotaryMaxDim / 2];
  const int tid = threadIdx.x, half = p.R / 2;
  const int blocks = (p.T + TB - 1) / TB;
  const int b = blockIdx.x / blocks, t0 = (blockIdx.x % blocks) * TB;
  const int nt = min(TB, p.T - t0);
  for (int i = tid; i < nt * half; i += 256) {
    const int t = i / half, j = i - t * half;
    cs[t * (kRotaryMaxDim / 2) + j] = rotary_turn(p, rotary_position(p, b, t0 + t), j);
  }
  __syncthreads();
  const int per = half + p.D - p.R, heads = p.H[0] + p.H[1];
  const int total = nt * heads * per;
  for (int i = tid; i < total; i += 256) {
    const int row = i / per, c = i - row * per;
    const int t = row / heads, hh = row - t * heads;
    const int w = hh >= p.H[0], h = w ? hh - p.H[0] : hh;
    const T* x = (const T*)p.x[w] + b * p.x_str[w][0] + h * p.x_str[w][1] + (t0 + t) * p.x_str[w][2];
    T* y = (T*)p.y[w] + b * p.y_str[w][0] + h * p.y_str[w][1] + (t0 + t) * p.y_str[w][2];
    if (c >= half) {
      y[half + c] = x[half + c];
      continue;
    }
    const int d0 = p.interleaved ? 2 * c : c, d1 = p.interleaved ? 2 * c + 1 : c + half;
    const float2 k = cs[t * (kRotaryMaxDim / 2) + c];
    const float u = (float)x[d0], v = (float)x[d1];
    y[d0] = (T)(u * k.x - v * k.y);
    y[d1] = (T)(v * k.x + u * k.y);
  }
}

template <typename T>
static void launch_rotary_t(const RotaryParams& p, bool chunks, hipStream_t stream) {
  auto go = [&](auto tb) {
    constexpr int TB = decltype(tb)::value;
    const dim3 grid((unsigned)((int64_t)p.B * ((p.T + TB - 1) / TB))), block(256);
    if (!chunks) hipLaunchKernelGGL((rotary_any_kernel<T, TB>), grid, block, 0, stream, p);
    else if (p.interleaved) hipLaunchKernelGGL((rotary_kernel<T, true, TB>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((rotary_kernel<T, false, TB>), grid, block, 0, stream, p);
  };
  // A token a block where there are few tokens, whose blocks run at once, else four.
  // us, one / four: 64 tokens of 40 heads of 128 in bf16 4.0 / 5.5, 1000 of 10 heads of 64
  // in fp32 4.8 / 4.6, 20000 of 8 heads of 128 23.4 / 16.1, 8192 of 40 heads in fp16
  // 31.9 / 30.4 (called in turn 39.0 / 35.0; all before put).
  if ((int64_t)p.B * p.T <= 512)
    go(std::integral_constant<int, 1>());
  else go(std::integral_constant<int, 4>());
}

void launch_rotary(const RotaryParams& p, int io_dtype, bool chunks, hipStream_t stream) {
  if (io_dtype == kF32) launch_rotary_t<float>(p, chunks, stream);
  else if (io_dtype == kF16) launch_rotary_t<f16>(p, chunks, stream);
  else launch_rotary_t<bf16>(p, chunks, stream);
}

}  // namespace nxa
