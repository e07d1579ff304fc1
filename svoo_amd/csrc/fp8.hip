// Quantising to 8 bits with a power-of-two scale per block of 128, and reading the values back.
//   e = min {e : amax 2^-e <= max(type)},  q = rne(x 2^-e),  scale byte e + 127 (e8m0)
// Blocks are 128 columns of one row, 128 rows x 128 columns, or (for products contracted over the rows) 128 rows of one
// column, written transposed.  Powers of two because the matrix instructions multiply them in at no cost, and exactly.
//
// What bounds it: memory.  Sixteen lanes hold a row's block, eight elements each: its maximum is four lane rotations.
// Where the transposed values are wanted too, a 128 x 128 tile is read once, stays in registers (8 rows x 8 columns a
// thread), and turns through LDS as bytes.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace svoo {

struct QuantArgs {
  const void* x;       // [rows][cols], x_row elements between rows
  int type;
  long long x_row;
  int rows, cols;
  int fp8;
  uint8_t* q;          // [rows][row_blocks * 128] or null
  uint8_t* scale;      // [row_blocks][rows], or [col_blocks][row_blocks] for square blocks
  uint8_t* qt;         // [cols][col_blocks * 128] or null
  uint8_t* scale_t;    // [col_blocks][cols], or [row_blocks][col_blocks]
  float* col_sums;     // [col_blocks][cols] or null
  int row_blocks, col_blocks;  // blocks of 128 columns in a row, of 128 rows in a column
};

template <int T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantArgs a) {
  constexpr int kUnroll = 4;
  const int t = threadIdx.x % 16;
  const unsigned units = (unsigned)a.rows * (unsigned)a.row_blocks, step = gridDim.x * 16;
  for (unsigned u0 = blockIdx.x * 16 + threadIdx.x / 16; u0 < units; u0 += step * kUnroll) {
    float f[kUnroll][8];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const unsigned u = u0 + i * step, row = u / a.row_blocks;
      const int col = (u - row * a.row_blocks) * 128 + t * 8;
      load_row8<T>(a.x, row * a.x_row + col, u < units ? a.cols - col : 0, f[i]);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const unsigned u = u0 + i * step;
      float amax = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(f[i][e]));
      const int e8 = block_exponent(max16(amax), a.fp8);
      if (u < units) {
        *(uint2*)(a.q + (size_t)u * 128 + t * 8) = quantize8(f[i], e8, a.fp8);
        if (t == 0) {
          const unsigned row = u / a.row_blocks;
          a.scale[(size_t)(u - row * a.row_blocks) * a.rows + row] = (uint8_t)(e8 + 127);
        }
      }
    }
  }
}

// One 128 x 128 tile per block.  Thread: columns (t % 16) 8 .. + 7 of rows (t / 16) 8 .. + 7.
// kSquare: one scale for the tile; else one per row (q) and one per column (qt).
template <int T, bool kSquare>
__global__ void __launch_bounds__(256) quantize_tile_kernel(QuantArgs a) {
  constexpr int kPitch = 33;  // dwords per transposed row
  __shared__ uint32_t turned[128 * kPitch];
  __shared__ float4 col_part[16][32];
  __shared__ float tile_part[4];
  __shared__ int col_exp[128];
  const int t = threadIdx.x % 16, g = threadIdx.x / 16;
  const int row0 = blockIdx.y * 128 + g * 8, col0 = blockIdx.x * 128 + t * 8;
  float f[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load_row8<T>(a.x, (long long)(row0 + i) * a.x_row + col0, row0 + i < a.rows ? a.cols - col0 : 0, f[i]);
  int tile_e = 0;
  if (kSquare) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(f[i][e]));
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if (threadIdx.x % kWave == 0) tile_part[threadIdx.x / kWave] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(tile_part[0], tile_part[1]), fmaxf(tile_part[2], tile_part[3]));
    tile_e = block_exponent(amax, a.fp8);
    if (threadIdx.x == 0) {
      if (a.scale != nullptr) a.scale[blockIdx.y * a.row_blocks + blockIdx.x] = (uint8_t)(tile_e + 127);
      if (a.scale_t != nullptr) a.scale_t[blockIdx.x * a.col_blocks + blockIdx.y] = (uint8_t)(tile_e + 127);
    }
  }
  if (a.q != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int e8 = tile_e;
      if (!kSquare) {
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(f[i][e]));
        e8 = block_exponent(max16(amax), a.fp8);
      }
      if (row0 + i < a.rows) {
        *(uint2*)(a.q + ((size_t)(row0 + i) * a.row_blocks + blockIdx.x) * 128 + t * 8) = quantize8(f[i], e8, a.fp8);
        if (!kSquare && t == 0) a.scale[(size_t)blockIdx.x * a.rows + row0 + i] = (uint8_t)(e8 + 127);
      }
    }
  }
  if (!kSquare && a.col_sums != nullptr) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[e] += f[i][e];
    }
    col_part[g][2 * t] = make_float4(s[0], s[1], s[2], s[3]);
    col_part[g][2 * t + 1] = make_float4(s[4], s[5], s[6], s[7]);
    __syncthreads();
    const int col = blockIdx.x * 128 + threadIdx.x;
    if (threadIdx.x < 128 && col < a.cols) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) v += ((const float*)col_part[k])[threadIdx.x];
      a.col_sums[(size_t)blockIdx.y * a.cols + col] = v;
    }
    __syncthreads();
  }
  if (a.qt == nullptr) return;
  int ce[8];
  if (kSquare) {
#pragma unroll
    for (int e = 0; e < 8; ++e) ce[e] = tile_e;
  } else {
    float m[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m[e] = fmaxf(m[e], finite_abs(f[i][e]));
    }
    col_part[g][2 * t] = make_float4(m[0], m[1], m[2], m[3]);
    col_part[g][2 * t + 1] = make_float4(m[4], m[5], m[6], m[7]);
    __syncthreads();
    if (threadIdx.x < 128) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) v = fmaxf(v, ((const float*)col_part[k])[threadIdx.x]);
      const int e8 = block_exponent(v, a.fp8), col = blockIdx.x * 128 + threadIdx.x;
      col_exp[threadIdx.x] = e8;
      if (col < a.cols) a.scale_t[(size_t)blockIdx.y * a.cols + col] = (uint8_t)(e8 + 127);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) ce[e] = col_exp[t * 8 + e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i][e];
    const uint2 w = quantize8(v, ce[e], a.fp8);
    turned[(t * 8 + e) * kPitch + g * 2] = w.x;
    turned[(t * 8 + e) * kPitch + g * 2 + 1] = w.y;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = i * 32 + threadIdx.x / 8, part = threadIdx.x % 8, col = blockIdx.x * 128 + c;
    const uint32_t* p = turned + c * kPitch + part * 4;
    if (col < a.cols)
      *(u32x4_t*)(a.qt + ((size_t)col * a.col_blocks + blockIdx.y) * 128 + part * 16) = u32x4_t{p[0], p[1], p[2], p[3]};
  }
}

// Column sums of the tiles to one row: 64 columns a block, 16 slices of the tiles, in a fixed order.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, int parts, int cols, void* out,
                                                          int type) {
  __shared__ float sums[16][kWave];
  const int col = blockIdx.x * kWave + threadIdx.x % kWave, slice = threadIdx.x / kWave;
  float s = 0.0f;
  if (col < cols) {
#pragma unroll 8
    for (int i = slice; i < parts; i += 16) s += part[(size_t)i * cols + col];
  }
  sums[slice][threadIdx.x % kWave] = s;
  __syncthreads();
  if (slice != 0 || col >= cols) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sums[i][threadIdx.x];
  set_row_elem(out, type, col, s);
}

struct DequantArgs {
  const uint8_t* q;
  long long q_row;
  const uint8_t* scale;
  long long scale_row, scale_col;
  int tall;            // rows per scale
  int rows, cols, fp8;
  void* y;             // [rows][cols]
  int vecs;            // groups of eight columns
};

template <int T>
__global__ void __launch_bounds__(256) dequantize_kernel(DequantArgs a) {
  constexpr int kUnroll = 4;
  const unsigned total = (unsigned)a.rows * (unsigned)a.vecs, step = gridDim.x * 256;
  for (unsigned v0 = blockIdx.x * 256 + threadIdx.x; v0 < total; v0 += step * kUnroll) {
    uint2 w[kUnroll];
    int byte[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const unsigned v = min(v0 + i * step, total - 1), row = v / a.vecs;
      const int col = (v - row * a.vecs) * 8;
      w[i] = *(const uint2*)(a.q + row * a.q_row + col);
      byte[i] = a.scale[(row / a.tall) * a.scale_row + (col / 128) * a.scale_col];
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const unsigned v = v0 + i * step, row = v / a.vecs;
      const int col = (v - row * a.vecs) * 8;
      const float s = byte[i] == 255 ? __builtin_nanf("") : power2(byte[i] - 127);
      float f[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = (int)(h == 0 ? w[i].x : w[i].y);
        const f32x2_t lo = a.fp8 == kFp8E4m3 ? __builtin_amdgcn_cvt_pk_f32_fp8(d, false)
                                             : __builtin_amdgcn_cvt_pk_f32_bf8(d, false);
        const f32x2_t hi = a.fp8 == kFp8E4m3 ? __builtin_amdgcn_cvt_pk_f32_fp8(d, true)
                                             : __builtin_amdgcn_cvt_pk_f32_bf8(d, true);
        f[4 * h] = lo[0] * s;
        f[4 * h + 1] = lo[1] * s;
        f[4 * h + 2] = hi[0] * s;
        f[4 * h + 3] = hi[1] * s;
      }
      if (v < total) store_row8<T>(a.y, (long long)row * a.cols + col, a.cols - col, f);
    }
  }
}

template <class F>
static void for_type(int type, F f) {
  if (type == kRowBf16) f(std::integral_constant<int, kRowBf16>());
  else if (type == kRowF16) f(std::integral_constant<int, kRowF16>());
  else f(std::integral_constant<int, kRowF32>());
}

static int check_matrix(const char* name, int type, int fp8, long long rows, long long cols) {
  SVOO_REQUIRE(type >= 0 && type <= 2, SVOO_ERR_INVALID_ARG, "%s: element type %d (0 bf16, 1 fp16, 2 fp32)", name, type);
  SVOO_REQUIRE(fp8 == kFp8E4m3 || fp8 == kFp8E5m2, SVOO_ERR_INVALID_ARG, "%s: 8-bit type %d (0 e4m3, 1 e5m2)", name, fp8);
  SVOO_REQUIRE(rows >= 0 && cols > 0, SVOO_ERR_INVALID_ARG, "%s: %lld x %lld", name, rows, cols);
  SVOO_REQUIRE(rows <= 0x7fffff80ll && cols <= 0x7fffff80ll && (rows + 127) / 128 * ((cols + 127) / 128) < (1ll << 24),
               SVOO_ERR_UNSUPPORTED, "%s: %lld x %lld (fewer than 2^24 blocks of 128 x 128)", name, rows, cols);
  return SVOO_OK;
}

}  // namespace svoo

using namespace svoo;

extern "C" int svoo_fp8_quantize_rows(const void* x, int type, long long x_row_stride, long long rows, long long cols,
                                      int fp8_type, uint8_t* q, uint8_t* scale, void* stream) {
  static const char* name = "svoo_fp8_quantize_rows";
  if (const int rc = check_matrix(name, type, fp8_type, rows, cols)) return rc;
  if (rows == 0) return SVOO_OK;
  SVOO_REQUIRE(x && q && scale, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE((uintptr_t)q % 8 == 0, SVOO_ERR_INVALID_ARG, "%s: q must start at an 8-byte address", name);
  const int row_blocks = (int)((cols + 127) / 128);
  const QuantArgs a = {x, type, x_row_stride, (int)rows, (int)cols, fp8_type, q, scale, nullptr, nullptr, nullptr,
                       row_blocks, (int)((rows + 127) / 128)};
  const unsigned blocks = (unsigned)std::min((rows * row_blocks + 15) / 16, 4096ll);
  for_type(type, [&](auto t) {
    hipLaunchKernelGGL(quantize_rows_kernel<decltype(t)::value>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch(name);
}

extern "C" size_t svoo_fp8_quantize_tiles_workspace_size(long long rows, long long cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)((rows + 127) / 128) * (size_t)cols * sizeof(float);
}

extern "C" int svoo_fp8_quantize_tiles(const void* x, int type, long long x_row_stride, long long rows, long long cols,
                                       int fp8_type, int square, uint8_t* q, uint8_t* scale, uint8_t* qt,
                                       uint8_t* scale_t, void* col_sums, int col_sums_type, void* workspace,
                                       size_t ws_bytes, void* stream) {
  static const char* name = "svoo_fp8_quantize_tiles";
  if (const int rc = check_matrix(name, type, fp8_type, rows, cols)) return rc;
  SVOO_REQUIRE((uintptr_t)q % 8 == 0 && (uintptr_t)qt % 16 == 0, SVOO_ERR_INVALID_ARG,
               "%s: q and qt must start at 8 and 16-byte addresses", name);
  SVOO_REQUIRE(col_sums_type >= 0 && col_sums_type <= 2, SVOO_ERR_INVALID_ARG, "%s: element type %d", name, col_sums_type);
  SVOO_REQUIRE(!col_sums || !square, SVOO_ERR_INVALID_ARG, "%s: column sums of square blocks", name);
  SVOO_REQUIRE(rows > 0 || !col_sums, SVOO_ERR_INVALID_ARG, "%s: column sums of no rows", name);
  if (rows == 0) return SVOO_OK;
  SVOO_REQUIRE((q != nullptr) == (scale != nullptr) && (qt != nullptr) == (scale_t != nullptr), SVOO_ERR_INVALID_ARG,
               "%s: values without scales", name);
  SVOO_REQUIRE(x && (q || qt || col_sums), SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE(!col_sums || (workspace && ws_bytes >= svoo_fp8_quantize_tiles_workspace_size(rows, cols)),
               SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)", name, ws_bytes,
               svoo_fp8_quantize_tiles_workspace_size(rows, cols));
  const int row_blocks = (int)((cols + 127) / 128), col_blocks = (int)((rows + 127) / 128);
  SVOO_REQUIRE(col_blocks <= 65535, SVOO_ERR_UNSUPPORTED, "%s: %lld rows (8388480 at most)", name, rows);
  const QuantArgs a = {x,  type,    x_row_stride, (int)rows, (int)cols, fp8_type, q, scale, qt, scale_t,
                       col_sums ? (float*)workspace : nullptr, row_blocks, col_blocks};
  for_type(type, [&](auto t) {
    const dim3 grid(row_blocks, col_blocks), block(256);
    if (square)
      hipLaunchKernelGGL((quantize_tile_kernel<decltype(t)::value, true>), grid, block, 0, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL((quantize_tile_kernel<decltype(t)::value, false>), grid, block, 0, (hipStream_t)stream, a);
  });
  if (const int rc = check_launch(name)) return rc;
  if (!col_sums) return SVOO_OK;
  hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((cols + kWave - 1) / kWave)), dim3(1024), 0, (hipStream_t)stream,
                     (const float*)workspace, col_blocks, (int)cols, col_sums, col_sums_type);
  return check_launch(name);
}

extern "C" int svoo_fp8_dequantize(const uint8_t* q, long long q_row_stride, const uint8_t* scale,
                                   long long scale_row_stride, long long scale_col_stride, int rows_per_scale,
                                   long long rows, long long cols, int fp8_type, void* y, int type, void* stream) {
  static const char* name = "svoo_fp8_dequantize";
  if (const int rc = check_matrix(name, type, fp8_type, rows, cols)) return rc;
  SVOO_REQUIRE(rows_per_scale == 1 || rows_per_scale == 128, SVOO_ERR_INVALID_ARG, "%s: %d rows a scale (1 or 128)", name,
               rows_per_scale);
  if (rows == 0) return SVOO_OK;
  SVOO_REQUIRE(q && scale && y, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE((uintptr_t)q % 8 == 0 && q_row_stride % 8 == 0, SVOO_ERR_INVALID_ARG,
               "%s: rows of q must start at 8-byte addresses", name);
  const int vecs = (int)((cols + 7) / 8);
  SVOO_REQUIRE(rows * vecs < (1ll << 31), SVOO_ERR_UNSUPPORTED, "%s: %lld x %lld", name, rows, cols);
  const DequantArgs a = {q, q_row_stride, scale, scale_row_stride, scale_col_stride, rows_per_scale, (int)rows, (int)cols, fp8_type, y,
                         vecs};
  const unsigned blocks = (unsigned)std::min((rows * vecs + 255) / 256, 4096ll);
  for_type(type, [&](auto t) {
    hipLaunchKernelGGL(dequantize_kernel<decltype(t)::value>, dim3(blocks), dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch(name);
}
