// A gated residual and the layer norm behind it, with the backward pass.
//   forward   h = x + gate b, rounded to its type;  n = (h - mean) rstd;  y = n w + c  (modulated: w = 1 + scale, c = shift)
//   backward  g = dy w;  dt = dh + rstd (g - mean(g) - n mean(g n));  dx = dt;  db = dt gate;
//             dgate = sum_rows dt b,  dw = sum_rows dy n,  dc = sum_rows dy
// Without y (dy) it is the residual alone.  The statistics are of h as it is stored, so the backward pass reads h, not x.
// What bounds it: memory; forward reads x and b and writes h and y, backward reads dh, dy, h and b and writes dx and db.  A
// row stays in the registers of its lanes as it lies in memory; parameters lie in LDS, in fp32.
// bf16, modulated and gated: 32760 x 1536 82 us (4.9 TB/s) forward and 129 (4.7) backward, 75600 x 5120 625 (5.0) and 915 (5.1).
#include <algorithm>
#include <type_traits>

#include "colsums.h"

namespace svoo {

struct ResidualParam {
  const void* p;     // [cols] per batch entry, or null
  int type;
  long long batch;   // elements between batch entries (0: shared)
  float plus;        // added to its values
  float none;        // its value without one
};

struct ResidualArgs {
  const void* x;     // [batch][rows][cols], element strides (backward: null)
  long long x_batch, x_row;
  const void* b;
  long long b_batch, b_row;
  ResidualParam gate, w, c;
  void* h;           // contiguous (backward: read)
  void* y;           // contiguous or null
  float* mean;       // [batch * rows] or null
  float* rstd;
  const void* dh;    // backward, or null
  long long dh_batch, dh_row;
  const void* dy;    // or null
  long long dy_batch, dy_row;
  void* dx;          // contiguous or null
  void* db;
  float* partial;    // [blocks][3][cols] or null
  int want[3];       // sums of dgate, dw, dc
  unsigned rows, parts;
  int cols;
  float eps;
};

__device__ __forceinline__ float param_at(const ResidualParam& p, unsigned batch, int col) {
  return p.p != nullptr ? row_elem(p.p, p.type, batch * p.batch + col) + p.plus : p.none;
}

// A parameter of the block's batch entry into LDS, as lanes read it: four columns by chunk, half and lane.
template <int TPR, int NC>
__device__ __forceinline__ void stage_param(const ResidualParam& p, unsigned batch, int cols, f32x4_t* to) {
  for (int i = threadIdx.x; i < NC * TPR * 8; i += blockDim.x) {
    const int at = ((i / (TPR * 8) * 2 + i / 4 % 2) * TPR + i / 8 % TPR) * 4 + i % 4;
    ((float*)to)[at] = i < cols ? param_at(p, batch, i) : 0.0f;
  }
}

// What a type holds of eight values, as they lie in memory.
template <int T>
__device__ __forceinline__ void pack_row8(const float (&f)[8], u32x4_t (&v)[T == kRowF32 ? 2 : 1]) {
  if (T == kRowF32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[T == kRowF32 ? e / 4 : 0][e % 4] = __float_as_uint(f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[0][e] = T == kRowBf16 ? cvt_pk_bf16(f[2 * e], f[2 * e + 1])
                              : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * e]) |
                                    ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * e + 1]) << 16);
  }
}

template <int T, int TPR, int NC, bool kWhole>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) residual_fwd_kernel(ResidualArgs a) {
  // the widest rows' gate stays in memory: three parameters of 16384 columns are more than LDS holds
  constexpr bool kGateLds = NC * TPR * 8 * 12 <= 147456;
  __shared__ f32x4_t params[kGateLds ? 3 : 2][2 * NC * TPR];
  __shared__ float2 scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  const int groups = blockDim.x / TPR, t = threadIdx.x % TPR;
  const unsigned batch = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  stage_param<TPR, NC>(a.w, batch, a.cols, params[0]);
  stage_param<TPR, NC>(a.c, batch, a.cols, params[1]);
  if (kGateLds) stage_param<TPR, NC>(a.gate, batch, a.cols, params[kGateLds ? 2 : 0]);
  __syncthreads();
  const float inv = 1.0f / (float)a.cols;
  int half = 0;
  for (unsigned r = part * groups + threadIdx.x / TPR; r < a.rows; r += a.parts * groups) {
    int cols = a.cols;
    if (!kWhole) __asm__ volatile("" : "+s"(cols));  // masks of the row's end made here: held over the rows they spill
    const size_t row = (size_t)batch * a.rows + r;
    RawRow<T, NC> x;
    {
      RawRow<T, NC> b;
      x.template load<TPR, kWhole>(a.x, batch * a.x_batch + r * a.x_row, cols, t);
      b.template load<TPR, kWhole>(a.b, batch * a.b_batch + r * a.b_row, cols, t);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * TPR + t) * 8;
        float f[8];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          f32x4_t g;
          if (kGateLds) {
            g = params[kGateLds ? 2 : 0][(c * 2 + hh) * TPR + t];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = col + 4 * hh + e < cols ? param_at(a.gate, batch, col + 4 * hh + e) : 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) f[4 * hh + e] = fmaf(b.at(c, 4 * hh + e), g[e], x.at(c, 4 * hh + e));
        }
        pack_row8<T>(f, x.v[c]);  // past the row's end zeros
        if (kWhole ? col < cols : true) {
          // the packed values are stored as they are
          const int n = cols - col;
          const long long at = (long long)row * cols + col;
          if (T == kRowF32) {
            store_row8<T, kWhole>(a.h, at, n, f);
          } else if (n >= 8) {
            ((Dwords4*)((uint16_t*)a.h + at))->v = x.v[c][0];
          } else if (!kWhole) {
            store_row8_bits((uint16_t*)a.h + at, n, x.v[c][0]);
          }
        }
      }
    }
    if (a.y == nullptr) continue;  // uniform: all rows of a launch
    x.forget();
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
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + t) * 8;
      float y[8];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const f32x4_t wv = params[0][(c * 2 + hh) * TPR + t], cv = params[1][(c * 2 + hh) * TPR + t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[4 * hh + e] = fmaf((x.at(c, 4 * hh + e) - mean0 - dm) * rstd, wv[e], cv[e]);
          __asm__("" : "+v"(y[4 * hh + e]));  // an fp32 number in every kernel: some would round to fp16 in the same step
        }
      }
      store_row8<T, kWhole>(a.y, (long long)row * cols + col, cols - col, y);
    }
  }
}

template <int T, int TPR, int NC, bool kWhole>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) residual_bwd_kernel(ResidualArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, kGroups = kThreads / TPR;
  __shared__ f32x4_t params[2][2 * NC * TPR];
  __shared__ float2 scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  __shared__ float sums[kGroups > 1 ? (kGroups - 1) * TPR * 8 : 1];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const unsigned batch = blockIdx.x / a.parts, part = blockIdx.x % a.parts, step = a.parts * kGroups;
  stage_param<TPR, NC>(a.w, batch, a.cols, params[0]);
  stage_param<TPR, NC>(a.gate, batch, a.cols, params[1]);
  __syncthreads();
  const float inv = 1.0f / (float)a.cols;
  const bool normed = a.dy != nullptr, gated = a.want[0] != 0, has_dh = a.dh != nullptr;
  int half = 0;
  float dg[NC][8], dw[NC][8], dc[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[c][e] = dw[c][e] = dc[c][e] = 0.0f;
  const size_t row0 = (size_t)batch * a.rows;
  for (unsigned r = part * kGroups + group; r < a.rows; r += step) {
    RawRow<T, NC> h, dy, dh, b;
    const int cols = a.cols;
    float mean = 0.0f, rstd = 0.0f;
    if (has_dh) dh.template load<TPR, kWhole>(a.dh, batch * a.dh_batch + r * a.dh_row, cols, t);
    else dh.template load<TPR, kWhole>(a.h, 0, 0, t);  // zeros
    if (normed) {
      dy.template load<TPR, kWhole>(a.dy, batch * a.dy_batch + r * a.dy_row, cols, t);
      h.template load<TPR, kWhole>(a.h, (long long)(row0 + r) * cols, cols, t);
      mean = a.mean[row0 + r];
      rstd = a.rstd[row0 + r];
    } else {
      dy.template load<TPR, kWhole>(a.dh, 0, 0, t);
      h.template load<TPR, kWhole>(a.dh, 0, 0, t);
    }
    if (gated) b.template load<TPR, kWhole>(a.b, batch * a.b_batch + r * a.b_row, cols, t);
    else b.template load<TPR, kWhole>(a.dh, 0, 0, t);
    float s1 = 0.0f, s2 = 0.0f;
    if (normed) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const f32x4_t wv = params[0][(c * 2 + hh) * TPR + t];
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) {
            const int e = 4 * hh + e4;
            // past the row's end dy is 0, and so is whatever n enters
            const float n = (h.at(c, e) - mean) * rstd, d = dy.at(c, e), g = d * wv[e4];
            dc[c][e] += d;
            dw[c][e] = fmaf(d, n, dw[c][e]);
            s1 += g;
            s2 = fmaf(g, n, s2);
          }
        }
      h.forget();
      dy.forget();
      row_sums<TPR>(s1, s2, scratch, half);
      s1 *= inv;
      s2 *= inv;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * TPR + t) * 8;
      float dt[8], m[8];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const f32x4_t wv = params[0][(c * 2 + hh) * TPR + t], gv = params[1][(c * 2 + hh) * TPR + t];
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int e = 4 * hh + e4;
          const float n = (h.at(c, e) - mean) * rstd;
          dt[e] = normed ? fmaf(rstd, dy.at(c, e) * wv[e4] - s1 - n * s2, dh.at(c, e)) : dh.at(c, e);
          m[e] = dt[e] * gv[e4];
          dg[c][e] = fmaf(kWhole || col + e < cols ? dt[e] : 0.0f, b.at(c, e), dg[c][e]);
        }
      }
      const long long at = (long long)(row0 + r) * cols + col;
      if (a.dx != nullptr) store_row8<T, kWhole>(a.dx, at, cols - col, dt);
      if (a.db != nullptr) store_row8<T, kWhole>(a.db, at, cols - col, m);
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    if (!a.want[which]) continue;  // uniform
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = which == 0 ? dg[c][e] : which == 1 ? dw[c][e] : dc[c][e];
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
      if (group == 0)
        store_row8<kRowF32, kWhole>(a.partial, ((long long)blockIdx.x * 3 + which) * a.cols + col, a.cols - col, v);
    }
  }
}

template <class F>
static void for_residual_flag(bool v, F f) {
  if (v) f(std::true_type());
  else f(std::false_type());
}
template <class F>
static void for_residual_type(int type, F f) {
  if (type == kRowBf16) f(std::integral_constant<int, kRowBf16>());
  else if (type == kRowF16) f(std::integral_constant<int, kRowF16>());
  else f(std::integral_constant<int, kRowF32>());
}
// Lanes per row and chunks of eight elements a lane, from the row's width: a wave a row up to 1536 columns (32760 x 1536 84 us
// forward and 129 backward; four waves 124 and 132), four up to 6144 (75600 x 5120 627 and 915; sixteen 715 and 917).
template <class F>
static void for_residual_width(int cols, F f) {
  using std::integral_constant;
  if (cols <= 128) f(integral_constant<int, 16>(), integral_constant<int, 1>());
  else if (cols <= 512) f(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (cols <= 1536) f(integral_constant<int, 64>(), integral_constant<int, 3>());
  else if (cols <= 2048) f(integral_constant<int, 256>(), integral_constant<int, 1>());
  else if (cols <= 6144) f(integral_constant<int, 256>(), integral_constant<int, 3>());
  else if (cols <= 8192) f(integral_constant<int, 1024>(), integral_constant<int, 1>());
  else f(integral_constant<int, 1024>(), integral_constant<int, 2>());
}
static int row_groups(int cols) { return cols <= 128 ? 16 : cols <= 1536 ? 4 : 1; }

// Blocks that share a batch entry's rows in the backward pass, whose partial sums are joined at the end.
static unsigned residual_parts(long long batch, long long rows, int cols) {
  const long long groups = row_groups(cols);
  const long long most = std::max(512 / batch, 1ll), want = (rows + 4 * groups - 1) / (4 * groups);
  return (unsigned)std::min(most, std::max(want, 1ll));
}

static int check_residual(const char* name, int type, long long batch, long long rows, int cols) {
  SVOO_REQUIRE(type >= 0 && type <= 2, SVOO_ERR_INVALID_ARG, "%s: element type %d (0 bf16, 1 fp16, 2 fp32)", name, type);
  SVOO_REQUIRE(batch >= 0 && rows >= 0 && cols > 0, SVOO_ERR_INVALID_ARG, "%s: batch=%lld rows=%lld cols=%d", name, batch, rows,
               cols);
  SVOO_REQUIRE(cols <= 16384, SVOO_ERR_UNSUPPORTED, "%s: %d columns (1..16384)", name, cols);
  SVOO_REQUIRE(batch < (1ll << 31) && rows < (1ll << 31) && batch * rows < (1ll << 31), SVOO_ERR_UNSUPPORTED,
               "%s: 2^31 rows or more", name);
  // a block per batch entry at least, fewer than 2^32 threads in a launch, and a grid dimension of 2^16 for the joined sums
  SVOO_REQUIRE(batch < 65536, SVOO_ERR_UNSUPPORTED, "%s: %lld batch entries with parameters of their own (fewer than 65536)",
               name, batch);
  return SVOO_OK;
}
static bool elem_types_ok(int a, int b, int c) { return a >= 0 && a <= 2 && b >= 0 && b <= 2 && c >= 0 && c <= 2; }

}  // namespace svoo

using namespace svoo;

extern "C" int svoo_residual_norm_fwd(const void* x, int type, long long x_batch_stride, long long x_row_stride,
                                      const void* b, long long b_batch_stride, long long b_row_stride, const void* gate,
                                      int gate_type, long long gate_batch_stride, const void* w, int w_type,
                                      long long w_batch_stride, const void* c, int c_type, long long c_batch_stride,
                                      int modulated, float eps, long long batch, long long rows, int cols, void* h, void* y,
                                      float* mean, float* rstd, void* stream) {
  static const char* name = "svoo_residual_norm_fwd";
  if (const int rc = check_residual(name, type, batch, rows, cols)) return rc;
  SVOO_REQUIRE(elem_types_ok(gate_type, w_type, c_type), SVOO_ERR_INVALID_ARG,
               "%s: element types %d %d %d (0 bf16, 1 fp16, 2 fp32)", name, gate_type, w_type, c_type);
  if (batch * rows == 0) return SVOO_OK;
  SVOO_REQUIRE(x && b && h, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  ResidualArgs a = {};
  a.x = x;
  a.x_batch = x_batch_stride;
  a.x_row = x_row_stride;
  a.b = b;
  a.b_batch = b_batch_stride;
  a.b_row = b_row_stride;
  a.gate = {gate, gate_type, gate_batch_stride, 0.0f, 1.0f};
  a.w = {w, w_type, w_batch_stride, modulated ? 1.0f : 0.0f, 1.0f};
  a.c = {c, c_type, c_batch_stride, 0.0f, 0.0f};
  a.h = h;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = (unsigned)rows;
  a.cols = cols;
  a.eps = eps;
  for_residual_width(cols, [&](auto tpr, auto nc) {
    constexpr int kTpr = decltype(tpr)::value, kNc = decltype(nc)::value, kThreads = kTpr > 256 ? kTpr : 256;
    const long long groups = kThreads / kTpr, want = (rows + groups - 1) / groups;
    a.parts = (unsigned)std::min(want, std::max(std::max(512 / (kThreads / 256), 256) / batch, 1ll));
    for_residual_type(type, [&](auto t) {
      for_residual_flag(cols % 8 == 0, [&](auto whole) {
        hipLaunchKernelGGL((residual_fwd_kernel<decltype(t)::value, kTpr, kNc, decltype(whole)::value>),
                           dim3((unsigned)(batch * a.parts)), dim3(kThreads), 0, (hipStream_t)stream, a);
      });
    });
  });
  return check_launch(name);
}

extern "C" size_t svoo_residual_norm_bwd_workspace_size(long long batch, long long rows, int cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  return (size_t)batch * residual_parts(batch, rows, cols) * 3 * cols * sizeof(float);
}

extern "C" int svoo_residual_norm_bwd(const void* dh, long long dh_batch_stride, long long dh_row_stride, const void* dy,
                                      long long dy_batch_stride, long long dy_row_stride, int type, const void* h,
                                      const void* b, long long b_batch_stride, long long b_row_stride, const void* gate,
                                      int gate_type, long long gate_batch_stride, const void* w, int w_type,
                                      long long w_batch_stride, int modulated, const float* mean, const float* rstd,
                                      long long batch, long long rows, int cols, void* dx, void* db, void* dgate,
                                      int dgate_type, int dgate_per_batch, void* dw, int dw_type, int dw_per_batch, void* dc,
                                      int dc_type, int dc_per_batch, void* workspace, size_t ws_bytes, void* stream) {
  static const char* name = "svoo_residual_norm_bwd";
  if (const int rc = check_residual(name, type, batch, rows, cols)) return rc;
  SVOO_REQUIRE(elem_types_ok(gate_type, w_type, 0) && elem_types_ok(dgate_type, dw_type, dc_type), SVOO_ERR_INVALID_ARG,
               "%s: element types %d %d %d %d %d (0 bf16, 1 fp16, 2 fp32)", name, gate_type, w_type, dgate_type, dw_type, dc_type);
  const bool sums = dgate || dw || dc;
  if (batch * rows == 0) {
    SVOO_REQUIRE(!sums, SVOO_ERR_INVALID_ARG, "%s: parameter gradients of no rows", name);
    return SVOO_OK;
  }
  if (!dx && !db && !sums) return SVOO_OK;
  SVOO_REQUIRE(dh || dy, SVOO_ERR_INVALID_ARG, "%s: no incoming gradient", name);
  SVOO_REQUIRE(!dy || (h && mean && rstd), SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE(dy || (!dw && !dc), SVOO_ERR_INVALID_ARG, "%s: gradients of the norm's parameters without dy", name);
  SVOO_REQUIRE(!dgate || b, SVOO_ERR_INVALID_ARG, "%s: a gate's gradient without the branch", name);
  const size_t need = svoo_residual_norm_bwd_workspace_size(batch, rows, cols);
  SVOO_REQUIRE(!sums || (workspace && ws_bytes >= need), SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)", name,
               ws_bytes, need);
  ResidualArgs a = {};
  a.dh = dh;
  a.dh_batch = dh_batch_stride;
  a.dh_row = dh_row_stride;
  a.dy = dy;
  a.dy_batch = dy_batch_stride;
  a.dy_row = dy_row_stride;
  a.h = (void*)h;
  a.b = b;
  a.b_batch = b_batch_stride;
  a.b_row = b_row_stride;
  a.gate = {gate, gate_type, gate_batch_stride, 0.0f, 1.0f};
  a.w = {w, w_type, w_batch_stride, modulated ? 1.0f : 0.0f, 1.0f};
  a.mean = (float*)mean;
  a.rstd = (float*)rstd;
  a.dx = dx;
  a.db = db;
  a.partial = sums ? (float*)workspace : nullptr;
  a.want[0] = dgate != nullptr;
  a.want[1] = dw != nullptr;
  a.want[2] = dc != nullptr;
  a.rows = (unsigned)rows;
  a.parts = residual_parts(batch, rows, cols);
  a.cols = cols;
  for_residual_width(cols, [&](auto tpr, auto nc) {
    constexpr int kTpr = decltype(tpr)::value, kNc = decltype(nc)::value, kThreads = kTpr > 256 ? kTpr : 256;
    for_residual_type(type, [&](auto t) {
      for_residual_flag(cols % 8 == 0, [&](auto whole) {
        hipLaunchKernelGGL((residual_bwd_kernel<decltype(t)::value, kTpr, kNc, decltype(whole)::value>),
                           dim3((unsigned)(batch * a.parts)), dim3(kThreads), 0, (hipStream_t)stream, a);
      });
    });
  });
  if (const int rc = check_launch(name)) return rc;
  if (!sums) return SVOO_OK;
  const ColSumsArgs s = {(const float*)workspace, (unsigned)batch, a.parts, 3, cols, {dgate, dw, dc},
                         {dgate_type, dw_type, dc_type}, {!dgate_per_batch, !dw_per_batch, !dc_per_batch}};
  hipLaunchKernelGGL(column_sums_kernel, dim3((cols + kWave - 1) / kWave, 3, (unsigned)batch), dim3(1024), 0, (hipStream_t)stream, s);
  return check_launch(name);
}
