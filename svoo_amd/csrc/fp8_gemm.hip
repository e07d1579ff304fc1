// Product of 8-bit matrices with a power-of-two scale per block of 128 along the contracted dimension:
//   c[m][n] = act(sum_k 2^(ea[m][k/128]) a[m][k] 2^(eb[n or n/128][k/128]) b[n][k] + bias[n])
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies the scales in and accumulates in fp32.  A lane's 32 bytes of an operand
// may be any 32 of the 64 contracted positions as long as both operands agree, and one scale covers all of them.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace svoo {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

enum GemmAct { kActNone = 0, kActGeluTanh = 1 };

struct GemmArgs {
  const uint8_t* a;        // [m][kb * 128], a_row bytes between rows
  long long a_row;
  const uint8_t* a_scale;  // [m][kb]
  long long a_scale_row;
  const uint8_t* b;        // [n][kb * 128]
  long long b_row;
  const uint8_t* b_scale;  // [n >> b_shift][kb]
  long long b_scale_row;
  int b_shift;
  const void* bias;        // [n] or null
  int bias_type;
  int act;
  void* c;                 // [m][n]
  int c_type;
  int m, n, kb;
};

// Sums.  The 8-bit matrix instructions add eight products at a time, aligned to the largest and cut 13 bits below it,
// before they go to the fp32 accumulator (measured with powers of two; the same for the unscaled instructions): 3.5e-5 of
// a random sum's size, a sixth of the rounding to fp16 and a fiftieth of that to bf16.  A caller who asks for fp32 gets
// sums in fp32: the values widen to bf16 (exactly, scale included) and go through the bf16 instructions, which round
// nothing else, at half the rate.
template <int A>
__device__ __forceinline__ f32x16_t mfma_widened(i32x8_t a, i32x8_t b, f32x16_t c, int sa, int sb) {
  const float fa = __uint_as_float((uint32_t)sa << 23), fb = __uint_as_float((uint32_t)sb << 23);  // the exponent is read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bf16x8_t wa, wb;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bf16x2_t pa =
          A == kFp8E4m3
              ? (e % 2 == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[2 * i + e / 2], fa, false)
                            : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[2 * i + e / 2], fa, true))
              : (e % 2 == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(a[2 * i + e / 2], fa, false)
                            : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(a[2 * i + e / 2], fa, true));
      const bf16x2_t pb = e % 2 == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[2 * i + e / 2], fb, false)
                                     : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[2 * i + e / 2], fb, true);
      wa[2 * e] = pa[0];
      wa[2 * e + 1] = pa[1];
      wb[2 * e] = pb[0];
      wb[2 * e + 1] = pb[1];
    }
    c = mfma32x32x16(wa, wb, c);
  }
  return c;
}

template <int A>
__device__ __forceinline__ f32x16_t mfma_scaled(i32x8_t a, i32x8_t b, f32x16_t c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, A, 0, 0, sa, 0, sb);
}

__device__ __forceinline__ float activation(float v, int act) {
  if (act == kActGeluTanh) {
    // v (1 + tanh(u)) / 2 = v / (1 + exp(-2u)),  u = sqrt(2 / pi) (v + 0.044715 v^3)
    const float u = 1.5957691216057308f * fmaf(0.044715f * v * v, v, v);
    return v / (1.0f + expf(-u));
  }
  return v;
}

template <int A, bool kWide>
__global__ void __launch_bounds__(256) fp8_gemm_kernel(GemmArgs g) {
  __shared__ u32x4_t lds[2][128 * 8];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int m0 = blockIdx.y * 128, n0 = blockIdx.x * 128;
  const int wm = (wave / 2) * 64, wn = (wave % 2) * 64, h = lane / 32, l = lane % 32;
  f32x16_t acc[2][2] = {};
  for (int kb = 0; kb < g.kb; ++kb) {
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int r = p * 32 + threadIdx.x / 8, c = threadIdx.x % 8;
      lds[0][r * 8 + (c ^ (r & 7))] = *(const u32x4_t*)(g.a + min(m0 + r, g.m - 1) * g.a_row + kb * 128 + c * 16);
      lds[1][r * 8 + (c ^ (r & 7))] = *(const u32x4_t*)(g.b + min(n0 + r, g.n - 1) * g.b_row + kb * 128 + c * 16);
    }
    __syncthreads();
    int sa[2], sb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sa[i] = g.a_scale[min(m0 + wm + i * 32 + l, g.m - 1) * g.a_scale_row + kb];
      sb[i] = g.b_scale[(min(n0 + wn + i * 32 + l, g.n - 1) >> g.b_shift) * g.b_scale_row + kb];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      i32x8_t fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ra = wm + i * 32 + l, rb = wn + i * 32 + l, c = 4 * j + 2 * h;
        const u32x4_t a0 = lds[0][ra * 8 + (c ^ (ra & 7))], a1 = lds[0][ra * 8 + ((c + 1) ^ (ra & 7))];
        const u32x4_t b0 = lds[1][rb * 8 + (c ^ (rb & 7))], b1 = lds[1][rb * 8 + ((c + 1) ^ (rb & 7))];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fa[i][e] = a0[e];
          fa[i][4 + e] = a1[e];
          fb[i][e] = b0[e];
          fb[i][4 + e] = b1[e];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[i][k] = kWide ? mfma_widened<A>(fa[i], fb[k], acc[i][k], sa[i], sb[k])
                                                    : mfma_scaled<A>(fa[i], fb[k], acc[i][k], sa[i], sb[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int n = n0 + wn + k * 32 + l;
    if (n >= g.n) continue;
    const float bias = g.bias != nullptr ? row_elem(g.bias, g.bias_type, n) : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = m0 + wm + i * 32 + (r / 4) * 8 + h * 4 + r % 4;
        if (m < g.m) set_row_elem(g.c, g.c_type, (long long)m * g.n + n, activation(acc[i][k][r] + bias, g.act));
      }
  }
}

}  // namespace svoo

using namespace svoo;

extern "C" size_t svoo_fp8_matmul_workspace_size(long long m, long long n, long long k) { return 0; }

extern "C" int svoo_fp8_matmul(const uint8_t* a, long long a_row_stride, const uint8_t* a_scale,
                               long long a_scale_row_stride, int a_type, const uint8_t* b, long long b_row_stride,
                               const uint8_t* b_scale, long long b_scale_row_stride, int b_rows_per_scale,
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
  SVOO_REQUIRE(m < (1ll << 30) && n < (1ll << 30) && k < (1ll << 30), SVOO_ERR_UNSUPPORTED, "%s: m=%lld n=%lld k=%lld", name,
               m, n, k);
  if (m == 0 || n == 0) return SVOO_OK;
  SVOO_REQUIRE(a && a_scale && b && b_scale && c, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE(((uintptr_t)a | (uintptr_t)b) % 16 == 0 && (a_row_stride | b_row_stride) % 16 == 0, SVOO_ERR_INVALID_ARG,
               "%s: rows must start at 16-byte addresses", name);
  const GemmArgs g = {a, a_row_stride, a_scale, a_scale_row_stride, b, b_row_stride, b_scale, b_scale_row_stride,
                      b_rows_per_scale == 128 ? 7 : 0, bias, bias_type, act, c, c_type, (int)m, (int)n, (int)(k / 128)};
  const dim3 grid((unsigned)((n + 127) / 128), (unsigned)((m + 127) / 128));
  auto launch = [&](auto type, auto wide) {
    hipLaunchKernelGGL((fp8_gemm_kernel<decltype(type)::value, decltype(wide)::value>), grid, dim3(256), 0,
                       (hipStream_t)stream, g);
  };
  auto launch_type = [&](auto type) {
    if (c_type == kRowF32) launch(type, std::true_type());
    else launch(type, std::false_type());
  };
  if (a_type == kFp8E4m3) launch_type(std::integral_constant<int, kFp8E4m3>());
  else launch_type(std::integral_constant<int, kFp8E5m2>());
  return check_launch(name);
}
