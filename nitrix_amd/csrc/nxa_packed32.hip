// Packed-sequence attention in fp32: the kernels of nxa_attn32.hip on one
// sequence at a time (nxa_packed.h).
#define NXA_PACKED 1
#include "nxa_attn32.hip"

namespace nxa {

// Per row: -delta = -sum_d O dO and -lse log2(e); 16 lanes a row.  (Rows of
// no sequence get a value that nothing reads.)
__global__ __launch_bounds__(256) void packed_delta32_kernel(const PackedParams p) {
  const int64_t rows = (int64_t)p.Hk * p.G * p.T;
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  float acc = 0.f;
  if (row < rows) {
    const int64_t h = row / p.T, t = row % p.T;
    const float* o = (const float*)p.o + h * p.o_str[1] + t * p.o_str[2];
    const float* d = (const float*)p.dout + h * p.do_str[1] + t * p.do_str[2];
    for (int c = sub * 4; c < p.Dv; c += 64) {
      const f32x4 x = ld16(o + c), y = ld16(d + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc += x[j] * y[j];
    }
  }
  acc += __shfl_xor(acc, 8, 16);
  acc += __shfl_xor(acc, 4, 16);
  acc += __shfl_xor(acc, 2, 16);
  acc += __shfl_xor(acc, 1, 16);
  if (row < rows && sub == 0) {
    p.ndelta[row] = -acc;
    p.nlse2[row] = -p.lse[row] * kLog2e;
  }
}

// Head dim 64: the kernels whose four waves share 32 rows and split the
// streamed tiles, against 128 rows a block and 32 a wave.  The first have four
// times the blocks and waste fewer rows at a sequence's end, the second read
// every tile once for four waves.  By 128-row blocks and tokens a sequence,
// 8 heads on 2 unless said, us of the pass, large block -> change with the
// split one: forward, 192 blocks (6 heads) of one sequence of 4096 1430 - 59,
// causal 1487 - 159; 256 blocks 1434 + 16, sequences of 512 225 + 33; 20 volumes
// of 250 tokens (235 blocks) 352 - 8.  dQ: 256 blocks, 512 tokens 225 - 4, causal
// 224 - 19, 4096 1434 - 52, causal 1495 - 251; 1024 blocks, 512 tokens 760 + 19,
// 2048 2737 - 17, causal 1589 - 43; volumes 352 - 49.  dK / dV: 64 blocks 374 -
// 94; 256 blocks, all keys, 512 tokens 225 + 19, 4096 1434 + 57, causal 224 - 9,
// 1495 - 306; volumes 352 - 15; 1024 blocks, causal 531 + 93.
// Between the counts (8 heads of their own keys, sequences of one length, us of
// the pass, split / large).  Forward, 256 tokens a sequence: 96 blocks 21 / 25,
// 160 31 / 26, 200 59 / 52, 224 39 / 26, 240 40 / 27, 288 49 / 44; some 1100
// tokens: 96 75 / 123, 160 95 / 104, 200 121 / 90, 224 122 / 101, 240 123 / 105,
// 288 152 / 168; the same causal 40 / 123, 59 / 104, 68 / 88, 78 / 98, 83 / 104,
// 94 / 102.  Backward, all keys, the rule of dK / dV alone changed: 144 blocks
// of 192 tokens 94 / 93, 329 123 / 111; 176 of 201 105 / 93, 352 129 / 113; 208 of
// 195 110 / 136, 256 112 / 94, 332 145 / 123; 240 of 192 112 / 117, 256 114 / 96,
// 320 146 / 167, 426 180 / 219.  So from 130 to 240 blocks sequences that are all
// short or all alike lose to the large forward block, by up to 17 us; where their
// lengths differ (the volumes above, the usual call) the split one gains, and
// the host does not know the lengths.  The 320 tokens of dK / dV lie among
// crossings that move with the rounding up to whole blocks and rounds.
static int64_t blocks128(const PackedParams& p, int heads) { return (int64_t)heads * p.T / 128; }
static bool split_fwd(const PackedParams& p) { return blocks128(p, p.Hk * p.G) < 240; }
static bool split_dq(const PackedParams& p) {
  const int64_t n = blocks128(p, p.Hk * p.G);
  return n <= 512 || (n <= 1024 && p.T / p.nseq >= 2048);
}
static bool split_dkdv(const PackedParams& p) {
  const int64_t n = blocks128(p, p.Hk * p.parts);
  return n <= 128 || (n <= 256 && (p.causal || p.T / p.nseq < 320));
}

int64_t packed_fwd32_threads(const PackedParams& p, int dp) {
  return packed_threads(p, (int64_t)p.Hk * p.G, dp == 64 && split_fwd(p) ? 32 : 128, 256);
}
int64_t packed_bwd32_threads(const PackedParams& p, int dp) {
  const int64_t delta = ((int64_t)p.Hk * p.G * p.T + 15) / 16 * 256;
  const int64_t q = (int64_t)p.Hk * p.G, k = (int64_t)p.Hk * p.parts;
  const int64_t dq = packed_threads(p, q, dp == 64 && split_dq(p) ? 32 : 128, 256);
  const int64_t dkdv = packed_threads(p, k, dp == 64 && split_dkdv(p) ? 32 : 128, 256);
  const int64_t most = dq > dkdv ? dq : dkdv;
  return delta > most ? delta : most;
}

template <int DP, bool CA>
static void launch_packed_fwd32_t(PackedParams p, hipStream_t stream) {
  if constexpr (DP == 64) {
    if (split_fwd(p)) {
      p.slots = packed_slots(p, 32);
      p.nwork = p.Hk * p.G * p.slots;
      hipLaunchKernelGGL((fwd32s_kernel<false, CA>), dim3(p.nwork + kPackedZeroBlocks), dim3(256),
                         0, stream, p);
      return;
    }
  }
  p.slots = packed_slots(p, 128);
  p.nwork = p.Hk * p.G * p.slots;
  hipLaunchKernelGGL((fwd32_kernel<DP, false, CA>), dim3(p.nwork + kPackedZeroBlocks), dim3(256),
                     0, stream, p);
}

template <int DP, bool CA>
static void launch_packed_bwd32_t(PackedParams p, hipStream_t stream) {
  p.slots = packed_slots(p, 128);
  p.nwork = p.Hk * p.G * p.slots;
  const int64_t rows = (int64_t)p.Hk * p.G * p.T;
  hipLaunchKernelGGL(packed_delta32_kernel, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0,
                     stream, p);
  PackedParams s = p;  // over 32-row tiles
  s.slots = packed_slots(p, 32);
  s.nwork = p.Hk * p.G * s.slots;
  if constexpr (DP == 64) {
    if (split_dq(p))
      hipLaunchKernelGGL((dq32_kernel<DP, CA, true>), dim3(s.nwork + kPackedZeroBlocks), dim3(256),
                         0, stream, s);
    else
      hipLaunchKernelGGL((dq32_kernel<DP, CA>), dim3(p.nwork + kPackedZeroBlocks), dim3(256), 0,
                         stream, p);
    if (split_dkdv(p)) {
      hipLaunchKernelGGL((dkdv32_kernel<DP, CA, kF32Both, true>), dim3(p.Hk * p.parts * s.slots),
                         dim3(256), 0, stream, s);
      return;
    }
  } else {
    hipLaunchKernelGGL((dq32_kernel<DP, CA>), dim3(p.nwork + kPackedZeroBlocks), dim3(256), 0,
                       stream, p);
  }
  const dim3 grid(p.Hk * p.parts * p.slots);
  if constexpr (DP > 128) {
    hipLaunchKernelGGL((dkdv32_kernel<DP, CA, kF32Dv>), grid, dim3(256), 0, stream, p);
    hipLaunchKernelGGL((dkdv32_kernel<DP, CA, kF32Dk>), grid, dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((dkdv32_kernel<DP, CA>), grid, dim3(256), 0, stream, p);
  }
}

void launch_packed_fwd32(const PackedParams& p, int dp, hipStream_t stream) {
  auto go = [&](auto ca) {
    constexpr bool CA = decltype(ca)::value;
    if (dp == 64) launch_packed_fwd32_t<64, CA>(p, stream);
    else if (dp == 128) launch_packed_fwd32_t<128, CA>(p, stream);
    else launch_packed_fwd32_t<256, CA>(p, stream);
  };
  if (p.causal) go(std::true_type{});
  else go(std::false_type{});
}

void launch_packed_bwd32(const PackedParams& p, int dp, hipStream_t stream) {
  auto go = [&](auto ca) {
    constexpr bool CA = decltype(ca)::value;
    if (dp == 64) launch_packed_bwd32_t<64, CA>(p, stream);
    else if (dp == 128) launch_packed_bwd32_t<128, CA>(p, stream);
    else launch_packed_bwd32_t<256, CA>(p, stream);
  };
  if (p.causal) go(std::true_type{});
  else go(std::false_type{});
}

}  // namespace nxa
