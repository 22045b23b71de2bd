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
  hipLaunchKernelGGL((dkdv16_kernel<T, DP, false, CA, kDbNone>), dim3(p.Hk * p.slots), dim3(512),
                     0, stream, p);
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

void launch_packed_bwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream) {
  if (io_dtype == kF32) launch_packed_bwd32(p, dp, stream);
  else if (dp == 256) launch_packed_bwd16_wide(p, io_dtype, stream);
  else if (io_dtype == kF16) launch_packed_d<f16>(p, dp, stream);
  else launch_packed_d<bf16>(p, dp, stream);
}

}  // namespace nxa
