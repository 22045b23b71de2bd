// Packed-sequence forward (bf16 / fp16) at padded head dims 64 and 128, and
// the dispatch over types and head dims.  The kernel is that of nxa_fwd16.h
// on one sequence at a time; the mapping of its grid is in nxa_packed.h.
#define NXA_PACKED 1
#include "nxa_fwd16.h"

namespace nxa {

template <typename T, int DP, int NW>
static void launch_packed_t(PackedParams p, hipStream_t stream) {
  p.slots = packed_slots(p, NW * 32);
  p.nwork = p.Hk * p.G * p.slots;
  const dim3 grid(p.nwork + kPackedZeroBlocks), block(NW * 64);
  if (p.causal)
    hipLaunchKernelGGL((fwd16_kernel<T, DP, NW, kFbNone, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((fwd16_kernel<T, DP, NW, kFbNone, false>), grid, block, 0, stream, p);
}

template <typename T>
static void launch_packed_d(const PackedParams& p, int dp, hipStream_t stream) {
  if (dp == 64) launch_packed_t<T, 64, 8>(p, stream);
  else launch_packed_t<T, 128, 8>(p, stream);
}

void launch_packed_fwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream) {
  if (io_dtype == kF32) launch_packed_fwd32(p, dp, stream);
  else if (dp == 256) launch_packed_fwd16_wide(p, io_dtype, stream);
  else if (io_dtype == kF16) launch_packed_d<f16>(p, dp, stream);
  else launch_packed_d<bf16>(p, dp, stream);
}

}  // namespace nxa
