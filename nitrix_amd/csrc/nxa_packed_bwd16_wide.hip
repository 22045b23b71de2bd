// Packed-sequence backward (bf16 / fp16) at padded head dim 256, in a
// translation unit of its own for the compiler flags of nxa_bwd16_wide.hip.
#define NXA_PACKED 1
#include "nxa_bwd16.h"

namespace nxa {

template <typename T, bool CA>
static void launch_packed_wide_t(PackedParams p, hipStream_t stream) {
  p.slots = packed_slots(p, 128);
  p.nwork = p.Hk * p.G * p.slots;
  hipLaunchKernelGGL((dq16_kernel<T, 256, kFbNone, CA>), dim3(p.nwork + kPackedZeroBlocks),
                     dim3(256), 0, stream, p);
  hipLaunchKernelGGL((dkdv256_kernel<T, false, CA, kDbNone>), dim3(p.Hk * p.parts * p.slots),
                     dim3(256), 0, stream, p);
}

void launch_packed_bwd16_wide(const PackedParams& p, int io_dtype, hipStream_t stream) {
  if (io_dtype == kF16) {
    if (p.causal) launch_packed_wide_t<f16, true>(p, stream);
    else launch_packed_wide_t<f16, false>(p, stream);
  } else {
    if (p.causal) launch_packed_wide_t<bf16, true>(p, stream);
    else launch_packed_wide_t<bf16, false>(p, stream);
  }
}

}  // namespace nxa
