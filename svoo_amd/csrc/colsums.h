// Sums of partial rows into parameter gradients, in a fixed order.
#pragma once

#include "rows.h"

namespace svoo {

struct ColSumsArgs {
  const float* partial;  // [batch][parts][n_out][cols]
  unsigned batch, parts;
  int n_out, cols;
  void* out[3];          // [batch][cols], or [cols] where the sum is over the batch too; null: not wanted
  int type[3];
  int over_batch[3];
};

// 64 columns a block, 16 slices of the partial rows, added in order.
static __global__ void __launch_bounds__(1024) column_sums_kernel(ColSumsArgs a) {
  __shared__ float sums[16][kWave];
  const int col = blockIdx.x * kWave + threadIdx.x % kWave, slice = threadIdx.x / kWave, which = blockIdx.y;
  void* out = a.out[which];
  const bool all = a.over_batch[which] != 0;
  const unsigned entry = blockIdx.z, parts = all ? a.batch * a.parts : a.parts;
  if (out == nullptr || (all && entry != 0)) return;
  float s = 0.0f;
  if (col < a.cols) {
    const float* p = a.partial + ((size_t)entry * a.parts * a.n_out + which) * a.cols + col;
#pragma unroll 8
    for (unsigned i = slice; i < parts; i += 16) s += p[(size_t)i * a.n_out * a.cols];
  }
  sums[slice][threadIdx.x % kWave] = s;
  __syncthreads();
  if (slice != 0 || col >= a.cols) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
  set_row_elem(out, a.type[which], (long long)entry * a.cols + col, s);
}

}  // namespace svoo
