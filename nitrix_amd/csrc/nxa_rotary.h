// Parameter block and launcher of nxa_rotary.hip.
#pragma once

#include "nxa_common.h"

namespace nxa {

struct RotaryParams {
  const void* x[2];          // [B, H[i], T, D]
  void* y[2];
  int64_t x_str[2][3], y_str[2][3];  // batch, head, token (elements)
  int H[2];
  const void* positions;     // [B, T] int32 or int64
  int64_t pos_str[2];
  const double* freq;        // [R / 2] radians a position
  int B, T, D, R;
  int interleaved, inverse, pos64;
  float scale;
};

constexpr int kRotaryMaxDim = 256;
void launch_rotary(const RotaryParams& p, int io_dtype, bool chunks, hipStream_t stream);

}  // namespace nxa
