// Layer norm: the forward pass, the C entries.
#include "layernorm.h"

namespace svoo {

// What bounds it: memory.  16 lanes hold a row of up to 128 columns, a wave one of up to 10 chunks of 512, a block of 1024
// threads a wider one, as it lies in memory: the mean and the centred second moment are two passes over registers, and
// with 46 of them at 1536 columns eight waves a SIMD keep enough loads in flight.  A block's rows share a batch entry,
// whose parameters lie in LDS: in registers they would take more than the row, and loaded per row twice its bytes.
// Measured, modulated bf16: 32760 x 1536 36 us (5.6 TB/s; 66 us with parameters and the row's values in fp32 registers),
// 75600 x 5120 310 us (5.0 TB/s; 777 us); fp32 32760 x 1536 80 us (5.0 TB/s); to 8 bits 32760 x 1536 43 us (3.5 TB/s), bound
// by its arithmetic: vector instructions fill 84 of 104 thousand cycles, of the 16-bit form 55 of 95.
// Over other widths in whole chunks 3.7 to 5.2 TB/s (3.1 to 3.4 at 64 and 256); bf16 rows of an odd length, with no chunk
// on a 16-byte address, 2.8 to 4.5 TB/s (to 8 bits 1.8 to 3.9): the last chunk is loaded as the row's last eight and moved
// down (104816 x 2561 270 us; element by element, with a block per row, 587).
template <int T, int TPR, int NC, bool kWhole, bool kFp8>
__device__ __forceinline__ void norm_rows(const NormArgs& a, const f32x4_t* w, const f32x4_t* b, float2* scratch) {
  const int groups = blockDim.x / TPR, t = threadIdx.x % TPR;
  const unsigned batch = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const float inv = 1.0f / (float)a.cols;
  int half = 0;
  for (unsigned r = part * groups + threadIdx.x / TPR; r < a.rows_per_batch; r += a.parts * groups) {
    int cols = a.cols;
    if (!kWhole) __asm__ volatile("" : "+s"(cols));  // masks of the row's end made here: held over the rows they spill
    const size_t row = (size_t)batch * a.rows_per_batch + r;
    RawRow<T, NC> x;
    x.template load<TPR, kWhole>(a.x, batch * a.x_batch + r * a.x_row, cols, t);
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        s0 += x.at(c, e);
        s1 += x.at(c, e + 1);
      }
    s0 += s1;
    s1 = 0.0f;
    row_sums<TPR>(s0, s1, scratch, half);
    float mean0 = s0 * inv;
    __asm__("" : "+v"(mean0));  // rounded once: fused into some of the differences below it would not be the same in all
    x.forget();
    float d1 = 0.0f, d2 = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + t) * 8;
      float u1 = 0.0f, u2 = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = kWhole || col + e < cols ? x.at(c, e) - mean0 : 0.0f;
        u1 += d;
        u2 = fmaf(d, d, u2);
      }
      const bool in = !kWhole || col < cols;
      d1 += in ? u1 : 0.0f;
      d2 += in ? u2 : 0.0f;
    }
    row_sums<TPR>(d1, d2, scratch, half);
    // what the rounding of the mean left over: the deviations' own mean
    const float dm = d1 * inv, var = fmaf(-dm, dm, d2 * inv);
    const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);  // NaN stays
    if (t == 0) {
      if (a.mean != nullptr) a.mean[row] = fabsf(mean0) < __builtin_inff() ? mean0 + dm : mean0;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
    x.forget();
    const int blocks = (cols + 127) / 128;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + t) * 8;
      float y[8];
      bool in = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4_t wv = w[(c * 2 + h) * TPR + t], bv = b[(c * 2 + h) * TPR + t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[4 * h + e] = fmaf((x.at(c, 4 * h + e) - mean0 - dm) * rstd, wv[e], bv[e]);
          __asm__("" : "+v"(y[4 * h + e]));  // an fp32 number in every kernel: some would round to fp16 in the same step
        }
      }
      if (!kFp8) {
        store_row8_as<kWhole>(a.y, a.y_type, (long long)row * cols + col, cols - col, y);
      } else {
        // the row rounded to x's type, as a quantiser of the stored one would see it; 16 lanes hold a block of 128 columns
        round_row8<T>(y);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!kWhole || e == 0) in = col + e < cols;
          y[e] = in ? y[e] : 0.0f;
          amax = fmaxf(amax, fabsf(y[e]));
        }
        amax = max16(amax);
        if (!(amax < __builtin_inff())) {  // infinities do not count
          amax = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(y[e]));
          amax = max16(amax);
        }
        const int e8 = block_exponent(amax, a.fp8);
        if (col < blocks * 128) {
          *(uint2*)(a.q + (size_t)row * blocks * 128 + col) = quantize8(y, e8, a.fp8);
          if (t % 16 == 0) a.q_scale[(size_t)(col / 128) * a.rows + row] = (uint8_t)(e8 + 127);
        }
      }
    }
  }
}

template <int T, int TPR, int NC, bool kWhole, bool kFp8>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_fwd_kernel(NormArgs a) {
  __shared__ f32x4_t params[2][2 * NC * TPR];  // four columns each: chunk, half, lane
  __shared__ float2 scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  const unsigned batch = blockIdx.x / a.parts;
  for (int i = threadIdx.x; i < NC * TPR * 8; i += blockDim.x) {
    const int at = ((i / (TPR * 8) * 2 + i / 4 % 2) * TPR + i / 8 % TPR) * 4 + i % 4;
    const bool in = i < a.cols;
    ((float*)params[0])[at] = in && a.w != nullptr ? row_elem(a.w, a.w_type, batch * a.w_batch + i) + a.w_plus : 1.0f;
    ((float*)params[1])[at] = in && a.b != nullptr ? row_elem(a.b, a.b_type, batch * a.b_batch + i) : 0.0f;
  }
  __syncthreads();
  norm_rows<T, TPR, NC, kWhole, kFp8>(a, params[0], params[1], scratch);
}

// out[batch][col] = sum over parts of partial[batch][part][which][col]: 64 columns a block, 16 slices of the parts.
__global__ void __launch_bounds__(1024) norm_param_grad_kernel(const float* __restrict__ partial, unsigned parts, int cols,
                                                               void* dw, int dw_type, void* db, int db_type) {
  __shared__ float sums[16][kWave];
  const int col = blockIdx.x * kWave + threadIdx.x % kWave, slice = threadIdx.x / kWave;
  const int which = blockIdx.y;
  void* out = which == 0 ? dw : db;
  if (out == nullptr) return;
  float s = 0.0f;
  if (col < cols) {
    const float* p = partial + ((size_t)blockIdx.z * parts * 2 + which) * cols + col;
#pragma unroll 8
    for (unsigned i = slice; i < parts; i += 16) s += p[(size_t)i * 2 * cols];
  }
  sums[slice][threadIdx.x % kWave] = s;
  __syncthreads();
  if (slice != 0 || col >= cols) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
  set_row_elem(out, which == 0 ? dw_type : db_type, (long long)blockIdx.z * cols + col, s);
}

// Lanes per row and chunks of eight elements a lane, from the row's width; fewer classes for the slower rows that do not
// end with a chunk.
template <class F>
static void for_width(int cols, F f) {
  const bool whole = cols % 8 == 0;
  if (cols <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  else if (cols <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  else if (whole && cols <= 1024) f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
  else if (cols <= 1536) f(std::integral_constant<int, 64>(), std::integral_constant<int, 3>());
  else if (whole && cols <= 2560) f(std::integral_constant<int, 64>(), std::integral_constant<int, 5>());
  else if (cols <= 5120) f(std::integral_constant<int, 64>(), std::integral_constant<int, 10>());
  else if (cols <= 8192) f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>());
  else f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
}
template <class F>
static void for_type(int type, F f) {
  if (type == kRowBf16) f(std::integral_constant<int, kRowBf16>());
  else if (type == kRowF16) f(std::integral_constant<int, kRowF16>());
  else f(std::integral_constant<int, kRowF32>());
}

// Blocks that share a batch entry's rows in the backward pass: two per CU in all, eight or four where a lane has one chunk
// and registers for more waves, and no fewer than four rows a group where there are more.  bf16, two against eight or four:
// 256 columns 723 and 458 us, 512 424 and 360, 2048 403 and 311; with two chunks a lane 1024 columns 301 and 349.
static unsigned grad_parts(long long batch, long long rows_per_batch, int cols) {
  const long long groups = cols <= 128 ? 16 : cols <= 1536 ? 4 : 1;
  const long long most = std::max((cols <= 512 ? 2048 : cols > 1536 && cols <= 2048 ? 1024 : 512) / batch, 1ll), want = (rows_per_batch + 4 * groups - 1) / (4 * groups);
  return (unsigned)std::min(most, std::max(want, 1ll));
}

static int check_norm(const char* name, int x_type, long long batch, long long rows_per_batch, int cols, int threads) {
  SVOO_REQUIRE(x_type >= 0 && x_type <= 2, SVOO_ERR_INVALID_ARG, "%s: element type %d (0 bf16, 1 fp16, 2 fp32)", name,
               x_type);
  SVOO_REQUIRE(batch >= 0 && rows_per_batch >= 0 && cols > 0, SVOO_ERR_INVALID_ARG,
               "%s: batch=%lld rows=%lld cols=%d", name, batch, rows_per_batch, cols);
  SVOO_REQUIRE(cols <= 16384, SVOO_ERR_UNSUPPORTED, "%s: %d columns (1..16384)", name, cols);
  SVOO_REQUIRE(batch < (1ll << 31) && rows_per_batch < (1ll << 31) && batch * rows_per_batch < (1ll << 31),
               SVOO_ERR_UNSUPPORTED, "%s: 2^31 rows or more", name);
  // a block per batch entry at least, and fewer than 2^32 threads in a launch
  const long long most = (1ll << 32) / threads;
  SVOO_REQUIRE(batch < most, SVOO_ERR_UNSUPPORTED, "%s: %lld batch entries of %d columns (fewer than %lld)", name, batch, cols,
               most);
  return SVOO_OK;
}

}  // namespace svoo

using namespace svoo;

extern "C" int svoo_layer_norm_fwd(const void* x, int x_type, long long x_batch_stride, long long x_row_stride,
                                   const void* w, int w_type, long long w_batch_stride, const void* b, int b_type,
                                   long long b_batch_stride, int modulated, float eps, long long batch,
                                   long long rows_per_batch, int cols, void* y, int y_type, uint8_t* q, uint8_t* q_scale,
                                   int fp8_type, float* mean, float* rstd, void* stream) {
  static const char* name = "svoo_layer_norm_fwd";
  if (const int rc = check_norm(name, x_type, batch, rows_per_batch, cols, cols <= 5120 ? 256 : 1024)) return rc;
  SVOO_REQUIRE(w_type >= 0 && w_type <= 2 && b_type >= 0 && b_type <= 2 && y_type >= 0 && y_type <= 2,
               SVOO_ERR_INVALID_ARG, "%s: element types %d %d %d (0 bf16, 1 fp16, 2 fp32)", name, w_type, b_type, y_type);
  SVOO_REQUIRE(fp8_type == kFp8E4m3 || fp8_type == kFp8E5m2, SVOO_ERR_INVALID_ARG, "%s: 8-bit type %d (0 e4m3, 1 e5m2)",
               name, fp8_type);
  const long long rows = batch * rows_per_batch;
  if (rows == 0) return SVOO_OK;
  SVOO_REQUIRE((y != nullptr) != (q != nullptr) && (q != nullptr) == (q_scale != nullptr), SVOO_ERR_INVALID_ARG,
               "%s: one of y and (q, q_scale)", name);
  SVOO_REQUIRE((uintptr_t)q % 8 == 0, SVOO_ERR_INVALID_ARG, "%s: q must start at an 8-byte address", name);
  SVOO_REQUIRE(q == nullptr || y_type == x_type, SVOO_ERR_UNSUPPORTED, "%s: 8-bit rows of another type than x's", name);
  SVOO_REQUIRE(x, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  NormArgs a = {x, x_type, x_batch_stride, x_row_stride, w, b, w_batch_stride, b_batch_stride, w_type, b_type,
                modulated ? 1.0f : 0.0f, y, y_type, q, q_scale, fp8_type, mean, rstd, (unsigned)rows,
                (unsigned)rows_per_batch, 1, cols, eps};
  for_width(cols, [&](auto tpr, auto nc) {
    constexpr int kTpr = decltype(tpr)::value, kNc = decltype(nc)::value;
    constexpr int kThreads = kTpr > 256 ? kTpr : 256;
    // blocks that are resident (32 waves a CU at most), the rest of the rows in turn
    const long long groups = kThreads / kTpr, want = (rows_per_batch + groups - 1) / groups;
    a.parts = (unsigned)std::min(want, std::max(256 * (2048 / kThreads) / batch, 1ll));
    const dim3 grid((unsigned)(batch * a.parts)), block(kThreads);
    for_type(x_type, [&](auto type) {
      for_flag(cols % 8 == 0, [&](auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        if constexpr (kWhole || kNc == 1 || kNc == 3 || kNc == 10 || kTpr == 1024) {
          for_flag(q != nullptr, [&](auto to_fp8) {
            hipLaunchKernelGGL((norm_fwd_kernel<decltype(type)::value, kTpr, kNc, kWhole, decltype(to_fp8)::value>), grid,
                               block, 0, (hipStream_t)stream, a);
          });
        }
      });
    });
  });
  return check_launch(name);
}

extern "C" size_t svoo_layer_norm_bwd_workspace_size(long long batch, long long rows_per_batch, int cols) {
  if (batch <= 0 || rows_per_batch <= 0 || cols <= 0) return 0;
  const unsigned parts = grad_parts(batch, rows_per_batch, cols);
  return parts == 1 ? 0 : (size_t)batch * parts * 2 * cols * sizeof(float);
}

extern "C" int svoo_layer_norm_bwd(const void* x, int x_type, long long x_batch_stride, long long x_row_stride,
                                   const void* dy, int dy_type, long long dy_batch_stride, long long dy_row_stride,
                                   const void* w, int w_type, long long w_batch_stride, int modulated, const float* mean,
                                   const float* rstd, long long batch, long long rows_per_batch, int cols, void* dx,
                                   void* dw, int dw_type, void* db, int db_type, void* workspace, size_t ws_bytes,
                                   void* stream) {
  static const char* name = "svoo_layer_norm_bwd";
  if (const int rc = check_norm(name, x_type, batch, rows_per_batch, cols, cols <= 6144 ? 256 : 1024)) return rc;
  SVOO_REQUIRE(dy_type >= 0 && dy_type <= 2 && w_type >= 0 && w_type <= 2 && dw_type >= 0 && dw_type <= 2 &&
                   db_type >= 0 && db_type <= 2,
               SVOO_ERR_INVALID_ARG, "%s: element types %d %d %d %d (0 bf16, 1 fp16, 2 fp32)", name, dy_type, w_type,
               dw_type, db_type);
  if (batch == 0 || rows_per_batch == 0) {
    SVOO_REQUIRE(batch == 0 || (!dw && !db), SVOO_ERR_INVALID_ARG, "%s: parameter gradients of no rows", name);
    return SVOO_OK;
  }
  SVOO_REQUIRE(x && dy && mean && rstd, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  if (!dx && !dw && !db) return SVOO_OK;
  const unsigned parts = grad_parts(batch, rows_per_batch, cols);
  const bool joined = (dw || db) && parts > 1;
  SVOO_REQUIRE(!joined || (workspace && ws_bytes >= svoo_layer_norm_bwd_workspace_size(batch, rows_per_batch, cols)),
               SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)", name, ws_bytes,
               svoo_layer_norm_bwd_workspace_size(batch, rows_per_batch, cols));
  const NormGradArgs a = {x, x_type, x_batch_stride, x_row_stride, dy, dy_type, dy_batch_stride, dy_row_stride, w,
                          w_batch_stride, w_type, modulated ? 1.0f : 0.0f, mean, rstd, dx,
                          joined ? (float*)workspace : nullptr, joined ? nullptr : dw, joined ? nullptr : db, dw_type,
                          db_type, (unsigned)rows_per_batch, parts, cols};
  launch_norm_bwd(a, batch, (hipStream_t)stream);
  if (const int rc = check_launch(name)) return rc;
  if (!joined) return SVOO_OK;
  hipLaunchKernelGGL(norm_param_grad_kernel, dim3((cols + kWave - 1) / kWave, 2, (unsigned)batch), dim3(1024), 0,
                     (hipStream_t)stream, (const float*)workspace, parts, cols, dw, dw_type, db, db_type);
  return check_launch(name);
}
