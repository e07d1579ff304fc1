// Layer norm, plain, affine or modulated per batch entry, with its backward pass.
//   forward   n = (x - mean) rstd,  y = n w + b  (modulated: w = 1 + scale, b = shift of the row's batch entry)
//   backward  g = dy w,  dx = rstd (g - mean(g) - n mean(g n)),  dw = sum_rows dy n,  db = sum_rows dy
// What bounds it: memory; forward reads x and writes y once, backward reads x and dy and writes dx once.  A row stays in
// the registers of its lanes as it lies in memory, eight consecutive elements per lane and chunk, so the mean and the
// centred second moment are passes over registers.  Statistics, sums and gradients are fp32.
#pragma once

#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace svoo {

struct NormArgs {
  const void* x;          // [batch][rows_per_batch][cols], element strides
  int x_type;
  long long x_batch, x_row;
  const void* w;          // weight or scale, [cols] per batch entry or null
  const void* b;          // bias or shift or null
  long long w_batch, b_batch;  // elements between batch entries (0: shared)
  int w_type, b_type;
  float w_plus;           // 1 for a scale
  void* y;                // [batch * rows_per_batch][cols] or null
  int y_type;
  uint8_t* q;             // 8-bit rows of padded columns or null
  uint8_t* q_scale;
  int fp8;
  float* mean;            // [batch * rows_per_batch] or null
  float* rstd;
  unsigned rows, rows_per_batch, parts;
  int cols;
  float eps;
};

struct NormGradArgs {
  const void* x;
  int x_type;
  long long x_batch, x_row;
  const void* dy;          // element strides
  int dy_type;
  long long dy_batch, dy_row;
  const void* w;
  long long w_batch;
  int w_type;
  float w_plus;
  const float* mean;
  const float* rstd;
  void* dx;                // [batch * rows_per_batch][cols], type of x, or null
  float* partial;          // [batch][parts][2][cols] or null (no parameter gradients)
  void* dw;                // with one part the sums go straight to the gradients
  void* db;
  int dw_type, db_type;
  unsigned rows_per_batch, parts;
  int cols;
};

template <class F>
static void for_flag(bool v, F f) {
  if (v) f(std::true_type());
  else f(std::false_type());
}

void launch_norm_bwd(const NormGradArgs& a, long long batch, hipStream_t s);  // layernorm_bwd.hip

}  // namespace svoo
