// Layer norm: the backward pass.
// Lanes keep their columns from row to row, so the column sums of dw and db stay in registers until the block's last row;
// they go to one partial row per block, which a second kernel adds in a fixed order: gradients do not depend on the
// schedule.  The next row is loaded while this one's two sums cross the lanes (and, for rows of several waves, a barrier).
// What bounds it: memory.  Measured, bf16 with parameter gradients: 75600 x 5120 510 us (4.6 TB/s of x, dy and dx; 1062 us
// with values in fp32 and no row ahead), fp32 32760 x 1536 132 us (4.6); 4.5 to 5.5 TB/s over widths of 128, 512, 1000 to 2048 and 4096 to 16384, 3.5 to
// 4.1 at 64, 256, 640 and 2560, where lanes are idle; rows of an odd length 2.1 to 4.3; fp32 rows above 8192 columns, whose
// column sums leave no registers for the row's, 2.7 to 3.1.
#include "layernorm.h"

namespace svoo {

template <int TX, int TD, int TPR, int NC, bool kWhole>
__device__ __forceinline__ void norm_grad_rows(const NormGradArgs& a, float (&dw)[NC][8], float (&db)[NC][8],
                                               float2* scratch) {
  const int groups = blockDim.x / TPR, t = threadIdx.x % TPR;
  const unsigned batch = blockIdx.x / a.parts, part = blockIdx.x % a.parts, step = a.parts * groups;
  const float inv = 1.0f / (float)a.cols;
  int half = 0;
  float w[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = (c * TPR + t) * 8 + e;
      w[c][e] = a.w != nullptr && col < a.cols ? row_elem(a.w, a.w_type, batch * a.w_batch + col) + a.w_plus : 1.0f;
    }
  unsigned r = part * groups + threadIdx.x / TPR;
  if (r >= a.rows_per_batch) return;  // all lanes of a row; for rows of several waves the whole block
  RawRow<TX, NC> x;
  RawRow<TD, NC> dy;
  const size_t row0 = (size_t)batch * a.rows_per_batch;
  float mean = a.mean[row0 + r], rstd = a.rstd[row0 + r];
  x.template load<TPR, kWhole>(a.x, batch * a.x_batch + r * a.x_row, a.cols, t);
  dy.template load<TPR, kWhole>(a.dy, batch * a.dy_batch + r * a.dy_row, a.cols, t);
  while (true) {
    constexpr bool kAhead = TPR < 1024;  // blocks of 1024 threads have 128 registers each
    const bool last = r + step >= a.rows_per_batch;
    RawRow<TX, NC> x1;
    RawRow<TD, NC> dy1;
    float mean1, rstd1;
    auto load_next = [&](unsigned next) __attribute__((always_inline)) {
      x1.template load<TPR, kWhole>(a.x, batch * a.x_batch + next * a.x_row, a.cols, t);
      dy1.template load<TPR, kWhole>(a.dy, batch * a.dy_batch + next * a.dy_row, a.cols, t);
      mean1 = a.mean[row0 + next];
      rstd1 = a.rstd[row0 + next];
    };
    if (kAhead) load_next(last ? r : r + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // past the row's end dy is 0, and so is whatever n enters
        const float n = (x.at(c, e) - mean) * rstd, d = dy.at(c, e), g = d * w[c][e];
        db[c][e] += d;
        dw[c][e] = fmaf(d, n, dw[c][e]);
        s1 += g;
        s2 = fmaf(g, n, s2);
      }
    x.forget();
    dy.forget();
    if (a.dx != nullptr) {
      row_sums<TPR>(s1, s2, scratch, half);
      s1 *= inv;
      s2 *= inv;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = (x.at(c, e) - mean) * rstd;
          v[e] = rstd * (dy.at(c, e) * w[c][e] - s1 - n * s2);
        }
        store_row8<TX, kWhole>(a.dx, (long long)(row0 + r) * a.cols + col, a.cols - col, v);
      }
    }
    if (last) break;
    r += step;
    if (!kAhead) load_next(r);
    x = x1;
    dy = dy1;
    mean = mean1;
    rstd = rstd1;
  }
}

template <int TX, int TD, int TPR, int NC, bool kWhole>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_bwd_kernel(NormGradArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kGroups = kThreads / TPR;
  __shared__ float2 scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  __shared__ float sums[kGroups > 1 ? (kGroups - 1) * TPR * 8 : 1];
  float dw[NC][8], db[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = db[c][e] = 0.0f;
  norm_grad_rows<TX, TD, TPR, NC, kWhole>(a, dw, db, scratch);
  if (a.partial == nullptr && a.dw == nullptr && a.db == nullptr) return;
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const unsigned batch = blockIdx.x / a.parts;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = which == 0 ? dw[c][e] : db[c][e];
      if (kGroups > 1) {  // the block's groups, in their order
        __syncthreads();
        if (group > 0)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[((group - 1) * 8 + e) * TPR + t] = v[e];
        __syncthreads();
        if (group == 0)
          for (int k = 0; k < kGroups - 1; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += sums[(k * 8 + e) * TPR + t];
      }
      const int col = (c * TPR + t) * 8;
      if (group != 0) continue;
      if (a.partial != nullptr)
        store_row8<kRowF32, kWhole>(a.partial, ((long long)blockIdx.x * 2 + which) * a.cols + col, a.cols - col, v);
      else if (which == 0 && a.dw != nullptr)
        store_row8_as<kWhole>(a.dw, a.dw_type, (long long)batch * a.cols + col, a.cols - col, v);
      else if (which == 1 && a.db != nullptr)
        store_row8_as<kWhole>(a.db, a.db_type, (long long)batch * a.cols + col, a.cols - col, v);
    }
  }
}

template <int TX, int TD, int TPR, int NC>
static void launch(const NormGradArgs& a, long long batch, hipStream_t s) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  for_flag(a.cols % 8 == 0, [&](auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    if constexpr (!kWhole || TX == TD)
      hipLaunchKernelGGL((norm_bwd_kernel<TX, TD, TPR, NC, kWhole>), dim3((unsigned)(batch * a.parts)), dim3(kThreads), 0, s,
                         a);
    else
      hipLaunchKernelGGL((norm_bwd_kernel<TX, TD, TPR, NC, false>), dim3((unsigned)(batch * a.parts)), dim3(kThreads), 0, s,
                         a);
  });
}

// Lanes per row and chunks of eight elements a lane, from the row's width (as grad_parts): the column sums of three chunks
// with two rows of x and dy fill 150 registers.  Gradients of another type than x's take fewer classes.
template <int TX, int TD>
static void launch_types(const NormGradArgs& a, long long batch, hipStream_t s) {
  const int cols = a.cols;
  if constexpr (TX == TD) {
    if (cols <= 128) return launch<TX, TD, 16, 1>(a, batch, s);
    if (cols <= 512) return launch<TX, TD, 64, 1>(a, batch, s);
    if (cols <= 1024) return launch<TX, TD, 64, 2>(a, batch, s);
  }
  if (cols <= 128) launch<TX, TD, 16, 1>(a, batch, s);
  else if (cols <= 1536) launch<TX, TD, 64, 3>(a, batch, s);
  else if (TX == TD && cols <= 2048) launch<TX, TX, 256, 1>(a, batch, s);
  else if (TX == TD && cols <= 4096) launch<TX, TX, 256, 2>(a, batch, s);
  else if (cols <= 6144) launch<TX, TD, 256, 3>(a, batch, s);
  else if (TX == TD && cols <= 8192) launch<TX, TX, 1024, 1>(a, batch, s);
  else launch<TX, TD, 1024, 2>(a, batch, s);
}

void launch_norm_bwd(const NormGradArgs& a, long long batch, hipStream_t s) {
  if (a.x_type == kRowBf16) {
    if (a.dy_type == kRowBf16) launch_types<kRowBf16, kRowBf16>(a, batch, s);
    else if (a.dy_type == kRowF16) launch_types<kRowBf16, kRowF16>(a, batch, s);
    else launch_types<kRowBf16, kRowF32>(a, batch, s);
  } else if (a.x_type == kRowF16) {
    if (a.dy_type == kRowBf16) launch_types<kRowF16, kRowBf16>(a, batch, s);
    else if (a.dy_type == kRowF16) launch_types<kRowF16, kRowF16>(a, batch, s);
    else launch_types<kRowF16, kRowF32>(a, batch, s);
  } else {
    if (a.dy_type == kRowBf16) launch_types<kRowF32, kRowBf16>(a, batch, s);
    else if (a.dy_type == kRowF16) launch_types<kRowF32, kRowF16>(a, batch, s);
    else launch_types<kRowF32, kRowF32>(a, batch, s);
  }
}

}  // namespace svoo
