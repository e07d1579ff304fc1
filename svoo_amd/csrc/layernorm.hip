// Layer norm, plain, affine or modulated per batch entry, with its backward pass.
//   forward   n = (x - mean) rstd,  y = n w + b  (modulated: w = 1 + scale, b = shift of the row's batch entry)
//   backward  g = dy w,  dx = rstd (g - mean(g) - n mean(g n)),  dw = sum_rows dy n,  db = sum_rows dy
//
// What bounds it: memory; forward reads x and writes y once, backward reads x and dy and writes dx once.  A row is held
// in the registers of TPR lanes, eight consecutive elements per lane and chunk, so the mean and the centred second
// moment are two passes over registers, not memory.  Lanes keep their columns from row to row: parameters are loaded
// once per wave (twice the row's own bytes if loaded per row) and the column sums of the backward pass stay in
// registers until the block's last row.  These go to one partial row per block and are added by a second kernel in a
// fixed order, so gradients do not depend on the schedule.  Statistics, sums and gradients are fp32.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace svoo {

struct NormArgs {
  const void* x;          // [batch][rows][cols], element strides
  int x_type;
  long long x_batch, x_row;
  const void* w;          // weight or scale, [cols] per batch entry or null
  const void* b;          // bias or shift or null
  long long w_batch, b_batch;  // elements between batch entries (0: shared)
  int w_type, b_type;
  float w_plus;           // 1 for a scale
  void* y;                // [batch * rows][cols] or null
  int y_type;
  uint8_t* q;             // 8-bit rows of padded columns or null
  uint8_t* q_scale;
  int fp8;
  float* mean;            // [batch * rows] or null
  float* rstd;
  unsigned rows, rows_per_batch;
  int cols;
  float eps;
};

// Sums of a and b over the TPR lanes of a row, in each of them.  For rows of several waves every thread of the block
// calls it; consecutive calls alternate between the two halves of scratch, so one barrier a call is enough.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float2* scratch, int& half) {
  if (TPR == 16) {
    a = sum16(a);
    b = sum16(b);
  } else {
    a = sum64(a);
    b = sum64(b);
    if (TPR > kWave) {
      constexpr int kWaves = TPR / kWave;
      float2* s = scratch + half * kWaves;
      half ^= 1;
      if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = make_float2(a, b);
      __syncthreads();
      a = b = 0.0f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        a += s[i].x;
        b += s[i].y;
      }
    }
  }
}

template <int TPR, int NC, bool kWhole>
__device__ __forceinline__ void load_params(const void* p, int type, long long at, float plus, float none, int cols, int t,
                                            float (&v)[NC][8]) {
  if (p != nullptr) load_row<TPR, NC, kWhole>(p, type, at, cols, t, v);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] = p != nullptr ? v[c][e] + plus : none;
}

template <int TPR, int NC, bool kWhole, bool kFp8>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_fwd_kernel(NormArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kGroups = kThreads / TPR;
  __shared__ float2 scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  int half = 0;
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.0f / (float)a.cols;
  float w[NC][8], b[NC][8];
  unsigned loaded = ~0u;
  for (unsigned row = blockIdx.x * kGroups + group; row < a.rows; row += gridDim.x * kGroups) {
    const unsigned batch = row / a.rows_per_batch;
    const long long at = batch * a.x_batch + (row - batch * a.rows_per_batch) * a.x_row;
    float x[NC][8];
    load_row<TPR, NC, kWhole>(a.x, a.x_type, at, a.cols, t, x);
    if (loaded != batch) {
      load_params<TPR, NC, kWhole>(a.w, a.w_type, batch * a.w_batch, a.w_plus, 1.0f, a.cols, t, w);
      load_params<TPR, NC, kWhole>(a.b, a.b_type, batch * a.b_batch, 0.0f, 0.0f, a.cols, t, b);
      loaded = batch;
    }
    float s = 0.0f, unused = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += x[c][e];
    row_sums<TPR>(s, unused, scratch, half);
    const float mean0 = s * inv;
    float d1 = 0.0f, d2 = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + t) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[c][e] = col + (kWhole ? 0 : e) < a.cols ? x[c][e] - mean0 : 0.0f;
        d1 += x[c][e];
        d2 = fmaf(x[c][e], x[c][e], d2);
      }
    }
    row_sums<TPR>(d1, d2, scratch, half);
    // what the rounding of the mean left over: the deviations' own mean
    const float dm = d1 * inv, rstd = 1.0f / sqrtf(fmaxf(fmaf(-dm, dm, d2 * inv), 0.0f) + a.eps);
    if (t == 0) {
      if (a.mean != nullptr) a.mean[row] = mean0 + dm;
      if (a.rstd != nullptr) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] = fmaf((x[c][e] - dm) * rstd, w[c][e], b[c][e]);
    if (!kFp8) {
      store_row<TPR, NC, kWhole>(a.y, a.y_type, (long long)row * a.cols, a.cols, t, x);
    } else {
      const int blocks = (a.cols + 127) / 128;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * 8;
        // the rounded row, as a quantiser of the stored one would see it; 16 lanes hold a block of 128 columns
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[c][e] = col + (kWhole ? 0 : e) < a.cols ? row_round(a.y_type, x[c][e]) : 0.0f;
          amax = fmaxf(amax, finite_abs(x[c][e]));
        }
        const int e8 = block_exponent(max16(amax), a.fp8);
        if (col < blocks * 128) {
          *(uint2*)(a.q + (size_t)row * blocks * 128 + col) = quantize8(x[c], e8, a.fp8);
          if (t % 16 == 0) a.q_scale[(size_t)(col / 128) * a.rows + row] = (uint8_t)(e8 + 127);
        }
      }
    }
  }
}

struct NormGradArgs {
  const void* x;
  int x_type;
  long long x_batch, x_row;
  const void* dy;          // element strides
  long long dy_batch, dy_row;
  int dy_type;
  const void* w;
  long long w_batch;
  int w_type;
  float w_plus;
  const float* mean;
  const float* rstd;
  void* dx;                // [batch * rows][cols], type of x, or null
  float* partial;          // [batch][parts][2][cols] or null (no parameter gradients)
  void* dw;                // with one part the sums go straight to the gradients
  void* db;
  int dw_type, db_type;
  unsigned rows_per_batch, parts;
  int cols;
};

template <int TPR, int NC, bool kWhole>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_bwd_kernel(NormGradArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kGroups = kThreads / TPR;
  __shared__ float2 scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  __shared__ float sums[kGroups > 1 ? (kGroups - 1) * TPR * 8 : 1];
  int half = 0;
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const unsigned batch = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const float inv = 1.0f / (float)a.cols;
  float w[NC][8], dw[NC][8], db[NC][8];
  load_params<TPR, NC, kWhole>(a.w, a.w_type, batch * a.w_batch, a.w_plus, 1.0f, a.cols, t, w);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = db[c][e] = 0.0f;
  for (unsigned r = part * kGroups + group; r < a.rows_per_batch; r += a.parts * kGroups) {
    const size_t row = (size_t)batch * a.rows_per_batch + r;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float n[NC][8], g[NC][8];
    float s1 = 0.0f, s2 = 0.0f;
    load_row<TPR, NC, kWhole>(a.x, a.x_type, batch * a.x_batch + r * a.x_row, a.cols, t, n);
    load_row<TPR, NC, kWhole>(a.dy, a.dy_type, batch * a.dy_batch + r * a.dy_row, a.cols, t, g);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[c][e] = (n[c][e] - mean) * rstd;  // past the row's end dy is 0, and so is whatever n enters
        db[c][e] += g[c][e];
        dw[c][e] = fmaf(g[c][e], n[c][e], dw[c][e]);
        g[c][e] *= w[c][e];
        s1 += g[c][e];
        s2 = fmaf(g[c][e], n[c][e], s2);
      }
    if (a.dx == nullptr) continue;
    row_sums<TPR>(s1, s2, scratch, half);
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) g[c][e] = rstd * (g[c][e] - s1 - n[c][e] * s2);
    store_row<TPR, NC, kWhole>(a.dx, a.x_type, (long long)row * a.cols, a.cols, t, g);
  }
  if (a.partial == nullptr && a.dw == nullptr && a.db == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float v[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = which == 0 ? dw[c][e] : db[c][e];
      if (kGroups > 1) {  // the block's groups, in their order
        __syncthreads();
        if (group > 0)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[((group - 1) * 8 + e) * TPR + t] = v[c][e];
        __syncthreads();
        if (group == 0)
          for (int k = 0; k < kGroups - 1; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] += sums[(k * 8 + e) * TPR + t];
      }
    }
    if (group != 0) continue;
    if (a.partial != nullptr)
      store_row<TPR, NC, kWhole>(a.partial, kRowF32, ((long long)blockIdx.x * 2 + which) * a.cols, a.cols, t, v);
    else if (which == 0 && a.dw != nullptr)
      store_row<TPR, NC, kWhole>(a.dw, a.dw_type, (long long)batch * a.cols, a.cols, t, v);
    else if (which == 1 && a.db != nullptr)
      store_row<TPR, NC, kWhole>(a.db, a.db_type, (long long)batch * a.cols, a.cols, t, v);
  }
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

// Lanes per row and chunks of eight elements a lane, from the row's width: rows up to 1536 columns fit one wave's
// registers (three chunks with their parameters and column sums, three waves per SIMD), wider ones a block.
template <class F>
static void for_width(int cols, F f) {
  if (cols <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
  else if (cols <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  else if (cols <= 1024) f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
  else if (cols <= 1536) f(std::integral_constant<int, 64>(), std::integral_constant<int, 3>());
  else if (cols <= 2048) f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
  else if (cols <= 4096) f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
  else if (cols <= 6144) f(std::integral_constant<int, 256>(), std::integral_constant<int, 3>());
  else if (cols <= 8192) f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>());
  else f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
}
template <class F>
static void for_flag(bool v, F f) {
  if (v) f(std::true_type());
  else f(std::false_type());
}

static int groups_for(int cols) { return cols <= 128 ? 16 : cols <= 1536 ? 4 : 1; }

// Blocks that share a batch entry's rows: two per CU in all, and no fewer than four rows a group where there are more.
static unsigned grad_parts(long long batch, long long rows_per_batch, int cols) {
  const long long groups = groups_for(cols);
  const long long most = std::max(512 / batch, 1ll), want = (rows_per_batch + 4 * groups - 1) / (4 * groups);
  return (unsigned)std::min(most, std::max(want, 1ll));
}

static int check_norm(const char* name, int x_type, long long batch, long long rows_per_batch, int cols) {
  SVOO_REQUIRE(x_type >= 0 && x_type <= 2, SVOO_ERR_INVALID_ARG, "%s: element type %d (0 bf16, 1 fp16, 2 fp32)", name,
               x_type);
  SVOO_REQUIRE(batch >= 0 && rows_per_batch >= 0 && cols > 0, SVOO_ERR_INVALID_ARG,
               "%s: batch=%lld rows=%lld cols=%d", name, batch, rows_per_batch, cols);
  SVOO_REQUIRE(cols <= 16384, SVOO_ERR_UNSUPPORTED, "%s: %d columns (1..16384)", name, cols);
  SVOO_REQUIRE(batch < (1ll << 31) && rows_per_batch < (1ll << 31) && batch * rows_per_batch < (1ll << 31),
               SVOO_ERR_UNSUPPORTED, "%s: 2^31 rows or more", name);
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
  if (const int rc = check_norm(name, x_type, batch, rows_per_batch, cols)) return rc;
  SVOO_REQUIRE(w_type >= 0 && w_type <= 2 && b_type >= 0 && b_type <= 2 && y_type >= 0 && y_type <= 2,
               SVOO_ERR_INVALID_ARG, "%s: element types %d %d %d (0 bf16, 1 fp16, 2 fp32)", name, w_type, b_type, y_type);
  SVOO_REQUIRE(fp8_type == kFp8E4m3 || fp8_type == kFp8E5m2, SVOO_ERR_INVALID_ARG, "%s: 8-bit type %d (0 e4m3, 1 e5m2)",
               name, fp8_type);
  const long long rows = batch * rows_per_batch;
  if (rows == 0) return SVOO_OK;
  SVOO_REQUIRE((y != nullptr) != (q != nullptr) && (q != nullptr) == (q_scale != nullptr), SVOO_ERR_INVALID_ARG,
               "%s: one of y and (q, q_scale)", name);
  SVOO_REQUIRE((uintptr_t)q % 8 == 0, SVOO_ERR_INVALID_ARG, "%s: q must start at an 8-byte address", name);
  SVOO_REQUIRE(x, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  const NormArgs a = {x,      x_type, x_batch_stride, x_row_stride, w,      b,  w_batch_stride, b_batch_stride, w_type,
                      b_type, modulated ? 1.0f : 0.0f, y,   y_type, q,  q_scale,        fp8_type,       mean,
                      rstd,   (unsigned)rows, (unsigned)rows_per_batch, cols, eps};
  for_width(cols, [&](auto tpr, auto nc) {
    constexpr int kTpr = decltype(tpr)::value, kNc = decltype(nc)::value, kThreads = kTpr > 256 ? kTpr : 256;
    const long long groups = kThreads / kTpr, cap = kTpr > 256 ? 512 : 2048;
    const dim3 grid((unsigned)std::min((rows + groups - 1) / groups, cap)), block(kThreads);
    for_flag(cols % 8 == 0, [&](auto whole) {
      for_flag(q != nullptr, [&](auto to_fp8) {
        hipLaunchKernelGGL((norm_fwd_kernel<kTpr, kNc, decltype(whole)::value, decltype(to_fp8)::value>), grid, block, 0,
                           (hipStream_t)stream, a);
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
  if (const int rc = check_norm(name, x_type, batch, rows_per_batch, cols)) return rc;
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
  const bool params = dw || db;
  const unsigned parts = grad_parts(batch, rows_per_batch, cols);
  const bool joined = params && parts > 1;
  SVOO_REQUIRE(!joined || (workspace && ws_bytes >= svoo_layer_norm_bwd_workspace_size(batch, rows_per_batch, cols)),
               SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)", name, ws_bytes,
               svoo_layer_norm_bwd_workspace_size(batch, rows_per_batch, cols));
  const NormGradArgs a = {x,       x_type, x_batch_stride, x_row_stride, dy,   dy_batch_stride, dy_row_stride,
                          dy_type, w,              w_batch_stride, w_type, modulated ? 1.0f : 0.0f, mean,
                          rstd,    dx,             joined ? (float*)workspace : nullptr, joined ? nullptr : dw,
                          joined ? nullptr : db, dw_type, db_type, (unsigned)rows_per_batch, parts, cols};
  for_width(cols, [&](auto tpr, auto nc) {
    constexpr int kTpr = decltype(tpr)::value, kNc = decltype(nc)::value, kThreads = kTpr > 256 ? kTpr : 256;
    for_flag(cols % 8 == 0, [&](auto whole) {
      hipLaunchKernelGGL((norm_bwd_kernel<kTpr, kNc, decltype(whole)::value>), dim3((unsigned)(batch * parts)),
                         dim3(kThreads), 0, (hipStream_t)stream, a);
    });
  });
  if (const int rc = check_launch(name)) return rc;
  if (!joined) return SVOO_OK;
  hipLaunchKernelGGL(norm_param_grad_kernel, dim3((cols + kWave - 1) / kWave, 2, (unsigned)batch), dim3(1024), 0,
                     (hipStream_t)stream, (const float*)workspace, parts, cols, dw, dw_type, db, db_type);
  return check_launch(name);
}
