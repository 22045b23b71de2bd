// Packed-sequence backward (bf16 / fp16) at padded head dims 64 and 128, and
// the dispatch over types and head dims.  The kernels are those of
// nxa_bwd16.h on one sequence at a time; dQ runs first and leaves the rows'
// -delta and -lse log2(e) for dK / dV.
#define NXA_PACKED 1
#include "nxa_bwd16.h"

namespace nxa {

template <typename T, int DP, bool CA>
static void launch_packed_t(PackedParams p, hipStream_t stream) {
  p.slots = packed_slots(p, 128);
  p.nwork = p.Hk * p.G * p.slots;
  hipLaunchKernelGGL((dq16_kernel<T, DP, kFbNone, CA>), dim3(p.nwork + kPackedZeroBlocks),
                     dim3(256), 0, stream, p);
  hipLaunchKernelGGL((dkdv16_kernel<T, DP, false, CA, kDbNone>), dim3(p.Hk * p.parts * p.slots),
                     dim3(512), 0, stream, p);
}

int64_t packed_bwd_threads(const PackedParams& p, int io_dtype, int dp) {
  if (io_dtype == kF32) return packed_bwd32_threads(p, dp);
  const int64_t dq = packed_threads(p, (int64_t)p.Hk * p.G, 128, 256);
  const int64_t dkdv = packed_threads(p, (int64_t)p.Hk * p.parts, 128, dp == 256 ? 256 : 512);
  return dq > dkdv ? dq : dkdv;
}

template <typename T>
static void launch_packed_d(const PackedParams& p, int dp, hipStream_t stream) {
  if (dp == 64) {
    if (p.causal) launch_packed_t<T, 64, true>(p, stream);
    else launch_packed_t<T, 64, false>(p, stream);
  } else {
    if (p.causal) launch_packed_t<T, 128, true>(p, stream);
    else launch_packed_t<T, 128, false>(p, stream);
  }
}

// Adds up the parts of dK (x = 0) and dV (x = 1), in order; rows of no
// sequence keep their zeros.
template <typename T>
__global__ __launch_bounds__(256) void packed_parts_kernel(const PackedParams p) {
  const bool is_v = blockIdx.y;
  const int n = is_v ? p.Dv : p.D;
  const float* part = p.dkv_part + (is_v ? (int64_t)p.parts * p.Hk * p.T * p.D : 0);
  const int64_t plane = (int64_t)p.Hk * p.T * n;
  const int lo = packed_offset(p, 0), hi = packed_offset(p, p.nseq);
  const int64_t hs = is_v ? p.dv_str[1] : p.dk_str[1], rs = is_v ? p.dv_str[2] : p.dk_str[2];
  T* out = (T*)(is_v ? p.dv : p.dk);
  typedef T t4 __attribute__((ext_vector_type(4)));
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < plane;
       i += (int64_t)gridDim.x * 1024) {
    const int64_t row = i / n;
    const int d = (int)(i - row * n), h = (int)(row / p.T), t = (int)(row - (int64_t)h * p.T);
    if (t < lo || t >= hi) continue;
    f32x4 x = *reinterpret_cast<const f32x4*>(part + i);
    for (int k = 1; k < p.parts; ++k) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(part + k * plane + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += y[e];
    }
    const t4 r = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    *reinterpret_cast<t4*>(out + h * hs + t * rs + d) = r;
  }
}

void launch_packed_parts(const PackedParams& p, int io_dtype, hipStream_t stream) {
  if (p.parts == 1) return;
  const int n = p.D > p.Dv ? p.D : p.Dv;
  const int64_t blocks = ((int64_t)p.Hk * p.T * n + 1023) / 1024;
  const dim3 grid((unsigned)(blocks < 2048 ? blocks : 2048), 2), block(256);
  if (io_dtype == kF32) hipLaunchKernelGGL(packed_parts_kernel<float>, grid, block, 0, stream, p);
  else if (io_dtype == kF16) hipLaunchKernelGGL(packed_parts_kernel<f16>, grid, block, 0, stream, p);
  else hipLaunchKernelGGL(packed_parts_kernel<bf16>, grid, block, 0, stream, p);
}

void launch_packed_bwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream) {
  if (io_dtype == kF32) launch_packed_bwd32(p, dp, stream);
  else if (dp == 256) launch_packed_bwd16_wide(p, io_dtype, stream);
  else if (io_dtype == kF16) launch_packed_d<f16>(p, dp, stream);
  else launch_packed_d<bf16>(p, dp, stream);
  launch_packed_parts(p, io_dtype, stream);
}

}  // namespace nxa
