// The product of 8-bit matrices: which kernel takes which sizes, the kernel for few rows, the sum over shares, the C entry.
#include "fp8_gemm.h"

namespace svoo {

// ---------------------------------------------------------------- few rows
// What bounds it: reading b once.  A block takes 32 rows of b (columns of c) and 32 rows of a, its waves every W-th block of
// 128 contracted positions, straight from memory into operands (nothing is used twice, so LDS would only add a trip): the
// lanes of a row's two halves take neighbouring 16-byte pieces.  The waves' sums meet in LDS, in the order of the waves.
template <int A, bool kWide>
__global__ void __launch_bounds__(1024) fp8_gemm_rows_kernel(GemmArgs g) {
  __shared__ __attribute__((aligned(16))) float part[16 * 32 * 32];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  const int l = lane % 32, h = lane / 32, m0 = blockIdx.y * 32, n0 = blockIdx.x * 32;
  const int m = min(m0 + l, g.m - 1), n = min(n0 + l, g.n - 1);
  const uint8_t* pa = g.a + m * g.a_row + h * 16;
  const uint8_t* pb = g.b + n * g.b_row + h * 16;
  const uint8_t* psa = g.a_scale + m * g.a_scale_row;
  const uint8_t* psb = g.b_scale + (n >> g.b_shift) * g.b_scale_row;
  f32x16_t acc = {};
  constexpr int kUnroll = 2;
  for (int k0 = wave; k0 < g.kb; k0 += waves * kUnroll) {
    i32x8_t a[kUnroll][2], b[kUnroll][2];
    int sa[kUnroll], sb[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = min(k0 + u * waves, g.kb - 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x4_t x = *(const u32x4_t*)(pb + k * 128ll + j * 32), y = *(const u32x4_t*)(pa + k * 128ll + j * 32);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          b[u][j / 2][j % 2 * 4 + e] = (int)x[e];
          a[u][j / 2][j % 2 * 4 + e] = (int)y[e];
        }
      }
      sa[u] = psa[k * g.a_scale_col];
      sb[u] = psb[k * g.b_scale_col];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (k0 + u * waves >= g.kb) break;  // uniform
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (kWide) {
          u32x4_t wa[4], wb[4];
          widen<A>(a[u][j], sa[u], wa);
          widen<kFp8E4m3>(b[u][j], sb[u], wb);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc = mfma32x32x16(as_bf16x8(wb[e]), as_bf16x8(wa[e]), acc);
        } else {
          acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[u][j], a[u][j], acc, 0, A, 0, sb[u], 0, sa[u]);
        }
      }
    }
  }
  // lane l: row l, columns 8 q + 4 h + e; a lane's pieces rotated by its row against bank conflicts
  if (m0 + l < g.m)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(f32x4_t*)(part + (wave * 32 + l) * 32 + (((2 * q + h) + l) & 7) * 4) =
          f32x4_t{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  for (int i = threadIdx.x; i < min(32, g.m - m0) * 32; i += blockDim.x) {
    const int r = i / 32, c = i % 32;
    if (n0 + c >= g.n) continue;
    const float* p = part + r * 32 + ((c / 4 + r) & 7) * 4 + c % 4;
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += p[w * 1024];
    if (g.bias != nullptr) s += row_elem(g.bias, g.bias_type, n0 + c);
    if (g.act == kActGeluTanh) s = gelu_exact(s);
    set_row_elem(g.c, g.c_type, (long long)(m0 + r) * g.n + n0 + c, s);
  }
}

// c = act(sum over shares + bias), in the order of the shares; four columns a thread.
__global__ void __launch_bounds__(256) fp8_gemm_join_kernel(GemmArgs g) {
  const unsigned quads = (g.n + 3) / 4, total = (unsigned)g.m * quads;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const unsigned m = i / quads;
    const int n = (int)(i - m * quads) * 4, count = min(4, g.n - n);
    const float* p = g.partial + (size_t)m * g.n + n;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = 0; k < g.splits; ++k, p += (size_t)g.m * g.n) {
      if (count == 4) {
        const u32x4_t v = ((const Dwords4*)p)->v;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += __uint_as_float(v[e]);
      } else {
        for (int e = 0; e < count; ++e) s[e] += p[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) {
        if (g.bias != nullptr) s[e] += row_elem(g.bias, g.bias_type, n + e);
        if (g.act == kActGeluTanh) s[e] = g.c_type == kRowF32 ? gelu_exact(s[e]) : gelu_fast(s[e]);
        set_row_elem(g.c, g.c_type, (long long)m * g.n + n + e, s[e]);
      }
  }
}

// ---------------------------------------------------------------- the choice
struct GemmPlan {
  int tile;    // 0: few rows
  int splits;
};

// The kernel and the number of shares with the shortest estimated time, in microseconds: rounds of items over the blocks
// that run at a time, each its stages and a constant for its start and end; shares add the partial sums' way out and back.
// Two blocks of 128 x 128 share a CU, and a round of no more than 256 has the CUs to itself.  Fitted to both tiles at 24
// sizes, e.g. (256 against 128) 2048 x 5120 x 5120 58 and 62 us, 4096 x 5120 x 5120 117 and 102, 32760 x 1536 x 8960 341 and
// 437, 2048 x 1536 x 8960 82 and 38; what it picks there is within a tenth of the faster.
static GemmPlan gemm_plan(long long m, long long n, long long kb, bool wide) {
  if (m <= 64) return {0, 1};
  GemmPlan best = {128, 1};
  double best_us = 1e30;
  for (int tile = wide ? 128 : 256; tile >= 128; tile -= 128) {
    const long long tiles = ((m + tile - 1) / tile) * ((n + tile - 1) / tile), blocks = gemm_blocks(tile);
    const double stage = tile == 256 ? 1.25 : wide ? 1.4 : 0.95, alone = tile == 256 || wide ? stage : 0.5;
    const double ends = tile == 256 ? 8.0 : 4.0;
    for (int splits = 1; splits <= 32 && (splits == 1 || kb / splits >= 2); ++splits) {
      const long long items = tiles * splits, left = items % blocks, stages = (kb + splits - 1) / splits;
      double us = (items / blocks) * (stages * stage + ends);
      if (left > 0) us += stages * (left <= 256 ? alone : stage) + ends;
      if (splits > 1) us += 5.0 + (double)m * n * splits * 8.0 / 6e6;
      if (us < best_us) {
        best_us = us;
        best = {tile, splits};
      }
    }
  }
  return best;
}

}  // namespace svoo

using namespace svoo;

extern "C" size_t svoo_fp8_matmul_workspace_size(long long m, long long n, long long k, int c_type) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const GemmPlan plan = gemm_plan(m, n, (k + 127) / 128, c_type == kRowF32);
  return plan.splits == 1 ? 0 : (size_t)plan.splits * (size_t)m * (size_t)n * sizeof(float);
}

extern "C" int svoo_fp8_matmul(const uint8_t* a, long long a_row_stride, const uint8_t* a_scale,
                               long long a_scale_row_stride, long long a_scale_col_stride, int a_type,
                               const uint8_t* b, long long b_row_stride, const uint8_t* b_scale,
                               long long b_scale_row_stride, long long b_scale_col_stride, int b_rows_per_scale,
                               const void* bias, int bias_type, int act, long long m, long long n, long long k, void* c,
                               int c_type, void* workspace, size_t ws_bytes, void* stream) {
  static const char* name = "svoo_fp8_matmul";
  SVOO_REQUIRE(a_type == kFp8E4m3 || a_type == kFp8E5m2, SVOO_ERR_INVALID_ARG, "%s: 8-bit type %d (0 e4m3, 1 e5m2)", name,
               a_type);
  SVOO_REQUIRE(bias_type >= 0 && bias_type <= 2 && c_type >= 0 && c_type <= 2, SVOO_ERR_INVALID_ARG,
               "%s: element types %d %d (0 bf16, 1 fp16, 2 fp32)", name, bias_type, c_type);
  SVOO_REQUIRE(b_rows_per_scale == 1 || b_rows_per_scale == 128, SVOO_ERR_INVALID_ARG, "%s: %d rows a scale (1 or 128)",
               name, b_rows_per_scale);
  SVOO_REQUIRE(act == kActNone || act == kActGeluTanh, SVOO_ERR_INVALID_ARG, "%s: activation %d", name, act);
  SVOO_REQUIRE(m >= 0 && n >= 0 && k > 0 && k % 128 == 0, SVOO_ERR_INVALID_ARG,
               "%s: m=%lld n=%lld k=%lld (k in whole blocks of 128)", name, m, n, k);
  if (m == 0 || n == 0) return SVOO_OK;
  SVOO_REQUIRE(a && a_scale && b && b_scale && c, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE(((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % 16 == 0 && (a_row_stride | b_row_stride) % 16 == 0,
               SVOO_ERR_INVALID_ARG, "%s: a, b and c must start at 16-byte addresses, and so the rows of a and b", name);
  SVOO_REQUIRE(a_row_stride >= k && b_row_stride >= k && a_scale_row_stride >= 0 && a_scale_col_stride >= 0 &&
                   b_scale_row_stride >= 0 && b_scale_col_stride >= 0,
               SVOO_ERR_INVALID_ARG, "%s: strides", name);
  // 32-bit offsets within a tile and within the scales
  const long long kb = k / 128, b_scales = b_rows_per_scale == 128 ? (n + 127) / 128 : n;
  SVOO_REQUIRE(m < (1ll << 28) && n < (1ll << 23) && a_row_stride < (1ll << 23) && b_row_stride < (1ll << 23),
               SVOO_ERR_UNSUPPORTED, "%s: m=%lld n=%lld, rows of %lld and %lld bytes", name, m, n, a_row_stride,
               b_row_stride);
  SVOO_REQUIRE(((m + 127) / 128) * ((n + 127) / 128) < (1ll << 25), SVOO_ERR_UNSUPPORTED, "%s: m=%lld n=%lld", name, m, n);
  SVOO_REQUIRE(a_scale_row_stride < (1ll << 31) && a_scale_col_stride < (1ll << 31) && b_scale_row_stride < (1ll << 31) &&
                   b_scale_col_stride < (1ll << 31) &&
                   (m + 255) * a_scale_row_stride + kb * a_scale_col_stride < (1ll << 31) &&
                   (b_scales + 255) * b_scale_row_stride + kb * b_scale_col_stride < (1ll << 31),
               SVOO_ERR_UNSUPPORTED, "%s: scales over 2^31 bytes", name);
  const bool wide = c_type == kRowF32;
  const GemmPlan plan = gemm_plan(m, n, kb, wide);
  const size_t need = svoo_fp8_matmul_workspace_size(m, n, k, c_type);
  SVOO_REQUIRE(need == 0 || (workspace && ws_bytes >= need), SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)",
               name, ws_bytes, need);
  const GemmArgs g = {a, a_row_stride, a_scale, a_scale_row_stride, a_scale_col_stride, b, b_row_stride, b_scale,
                      b_scale_row_stride, b_scale_col_stride, b_rows_per_scale == 128 ? 7 : 0, bias, bias_type, act, c,
                      c_type, (int)m, (int)n, (int)kb, plan.splits, (float*)workspace};
  hipStream_t s = (hipStream_t)stream;
  if (plan.tile == 0) {
    const dim3 grid((unsigned)((n + 31) / 32), (unsigned)((m + 31) / 32)), block(kWave * (unsigned)std::min(kb, 16ll));
    auto launch = [&](auto type, auto is_wide) {
      hipLaunchKernelGGL((fp8_gemm_rows_kernel<decltype(type)::value, decltype(is_wide)::value>), grid, block, 0, s, g);
    };
    auto launch_type = [&](auto type) {
      if (wide) launch(type, std::true_type());
      else launch(type, std::false_type());
    };
    if (a_type == kFp8E4m3) launch_type(std::integral_constant<int, kFp8E4m3>());
    else launch_type(std::integral_constant<int, kFp8E5m2>());
    return check_launch(name);
  }
  const int out = plan.splits == 1 ? c_type : wide ? kShareWide : kShare;
  if (plan.tile == 256 && !(a_type == kFp8E5m2 && act != kActNone && plan.splits == 1)) launch_gemm_256(g, a_type, out, s);
  else launch_gemm_128(g, a_type, out, s);
  if (const int rc = check_launch(name)) return rc;
  if (plan.splits == 1) return SVOO_OK;
  const long long threads = m * ((n + 3) / 4);
  hipLaunchKernelGGL(fp8_gemm_join_kernel, dim3((unsigned)std::min((threads + 255) / 256, 8192ll)), dim3(256), 0, s, g);
  return check_launch(name);
}
