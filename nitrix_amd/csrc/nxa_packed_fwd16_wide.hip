// Packed-sequence forward (bf16 / fp16) at padded head dim 256, in a
// translation unit of its own for the compiler flags of nxa_fwd16_wide.hip.
#define NXA_PACKED 1
#include "nxa_fwd16.h"

namespace nxa {

template <typename T>
static void launch_packed_wide_t(PackedParams p, hipStream_t stream) {
  p.slots = packed_slots(p, 128);
  p.nwork = p.Hk * p.G * p.slots;
  const dim3 grid(p.nwork + kPackedZeroBlocks), block(256);
  if (p.causal)
    hipLaunchKernelGGL((fwd16_kernel<T, 256, 4, kFbNone, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((fwd16_kernel<T, 256, 4, kFbNone, false>), grid, block, 0, stream, p);
}

void launch_packed_fwd16_wide(const PackedParams& p, int io_dtype, hipStream_t stream) {
  if (io_dtype == kF16) launch_packed_wide_t<f16>(p, stream);
  else launch_packed_wide_t<bf16>(p, stream);
}

}  // namespace nxa
