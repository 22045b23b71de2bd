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

template <int DP, bool CA>
static void launch_packed_fwd32_t(PackedParams p, hipStream_t stream) {
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
  hipLaunchKernelGGL((dq32_kernel<DP, CA>), dim3(p.nwork + kPackedZeroBlocks), dim3(256), 0,
                     stream, p);
  const dim3 grid(p.Hk * p.slots);
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
