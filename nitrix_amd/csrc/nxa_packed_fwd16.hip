// Packed-sequence forward (bf16 / fp16) at padded head dims 64 and 128, and
// the dispatch over types and head dims.  The kernel is that of nxa_fwd16.h
// on one sequence at a time; the mapping of its grid is in nxa_packed.h.
#define NXA_PACKED 1
#include "nxa_fwd16.h"

namespace nxa {

// The dense kernel's ring is a type of its own.
static_assert(FwdRing<128, 4, kFbNone, true>::NST == 2 &&
              FwdRing<128, 4, kFbNone, false>::NST == 4);

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

// Head dim 128: blocks of 4 waves and 128 rows (two a CU) or of 8 waves and
// 256 rows (whose pairs take turns at the matrix core).  The small block
// wastes fewer rows at a sequence's end and keys behind its diagonal, and has
// more blocks to fill the chip; the large one is faster once those do not
// matter.  bf16, 32 heads on 8, us of 8 against 4 waves: 16384 tokens, causal,
// sequences of 256 168 against 127, 1024 240 against 210, 2048 344 / 331, 4096
// 544 / 560, 16384 1852 / 1988; all keys, 512 205 / 187, 1024 310 / 300, 2048
// 515 / 533, 8192 1811 / 1973.  One sequence of 2048, 8 heads on 2 (64 large
// blocks): 51 / 41.  (At head dim 64 the small block is the faster one up to
// 4096 tokens a sequence by 1 to 38 %, and within 5 % from there on: it is
// always taken.)
static bool four_waves(const PackedParams& p) {
  if ((int64_t)p.Hk * p.G * (p.T / 256 + 1) < 256) return true;
  return p.T / p.nseq < (p.causal ? 3000 : 1400);
}

int64_t packed_fwd_threads(const PackedParams& p, int io_dtype, int dp) {
  if (io_dtype == kF32) return packed_fwd32_threads(p, dp);
  const int nw = dp == 128 && !four_waves(p) ? 8 : 4;
  return packed_threads(p, (int64_t)p.Hk * p.G, nw * 32, nw * 64);
}

template <typename T>
static void launch_packed_d(const PackedParams& p, int dp, hipStream_t stream) {
  if (dp == 64) launch_packed_t<T, 64, 4>(p, stream);
  else if (four_waves(p)) launch_packed_t<T, 128, 4>(p, stream);
  else launch_packed_t<T, 128, 8>(p, stream);
}

void launch_packed_fwd(const PackedParams& p, int io_dtype, int dp, hipStream_t stream) {
  if (io_dtype == kF32) launch_packed_fwd32(p, dp, stream);
  else if (dp == 256) launch_packed_fwd16_wide(p, io_dtype, stream);
  else if (io_dtype == kF16) launch_packed_d<f16>(p, dp, stream);
  else launch_packed_d<bf16>(p, dp, stream);
}

}  // namespace nxa
