// Product of 8-bit matrices with a power-of-two scale per block of 128 along the contracted dimension:
//   c[m][n] = act(sum_k 2^(ea[m][k/128]) a[m][k] 2^(eb[n or n/128][k/128]) b[n][k] + bias[n])
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies the scales in and accumulates in fp32.  A lane's 32 bytes of an operand
// may be any 32 of the 64 contracted positions as long as both operands agree, and one scale covers all of them.
#pragma once

#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace svoo {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

enum GemmAct { kActNone = 0, kActGeluTanh = 1, kActAny = 2 };
// Where a kernel takes the type of c, besides the row types: a share of the contracted dimension, by the 8-bit
// instructions or in fp32 throughout.
constexpr int kShare = 3, kShareWide = 4;

struct GemmArgs {
  const uint8_t* a;        // [m][kb * 128], a_row bytes between rows
  long long a_row;
  const uint8_t* a_scale;  // [m][kb]
  long long a_scale_row, a_scale_col;
  const uint8_t* b;        // [n][kb * 128]
  long long b_row;
  const uint8_t* b_scale;  // [n >> b_shift][kb]
  long long b_scale_row, b_scale_col;
  int b_shift;
  const void* bias;        // [n] or null
  int bias_type;
  int act;
  void* c;                 // [m][n]
  int c_type;
  int m, n, kb;
  int splits;              // shares of the contracted dimension, summed from partial [splits][m][n] afterwards
  float* partial;
};

// Sums.  The 8-bit matrix instructions add eight products at a time, aligned to the largest and cut 13 bits below it,
// before they go to the fp32 accumulator (measured with powers of two; the same for the unscaled instructions): 3.5e-5 of
// a random sum's size, a sixth of the rounding to fp16 and a fiftieth of that to bf16.  A caller who asks for fp32 gets
// sums in fp32: the values widen to bf16 (exactly, scale included) and go through the bf16 instructions, which round
// nothing else, at half the rate.
template <int T>
__device__ __forceinline__ void widen(i32x8_t v, int scale, u32x4_t (&out)[4]) {
  const float s = __uint_as_float((uint32_t)scale << 23);  // the instruction reads the exponent
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bf16x2_t lo, hi;
    if (T == kFp8E4m3) {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], s, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], s, true);
    } else {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v[i], s, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v[i], s, true);
    }
    out[i / 2][i % 2 * 2] = __builtin_bit_cast(uint32_t, lo);
    out[i / 2][i % 2 * 2 + 1] = __builtin_bit_cast(uint32_t, hi);
  }
}

// v sigmoid(2 u), u = sqrt(2 / pi) (v + 0.044715 v^3).
__device__ __forceinline__ float gelu_exact(float v) {
  return v / (1.0f + expf(-1.5957691216057308f * fmaf(0.044715f * v * v, v, v)));
}
// The same by the hardware's exp2 and reciprocal: a few 2^-22, for 16-bit results.
__device__ __forceinline__ float gelu_fast(float v) {
  const float e = __builtin_amdgcn_exp2f(v * fmaf(v * v, -0.10294323f, -2.3022082f));
  return v * __builtin_amdgcn_rcpf(1.0f + e);
}

// A 32 x 32 piece as 16 bits each: lane 16 b + 32 h + i gets columns 16 b + 8 h .. + 7 of row i in lo, of row 16 + i in hi.
template <int T>
__device__ __forceinline__ void pack_rows(const f32x16_t& c, u32x4_t& lo, u32x4_t& hi) {
  uint32_t w[8];  // columns 8 (i / 2) + 4 h + 2 (i % 2) and the next
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = T == kRowBf16 ? cvt_pk_bf16(c[2 * i], c[2 * i + 1])
                         : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)c[2 * i]) |
                               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)c[2 * i + 1]) << 16);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    // across the halves: columns 8 h .. + 7 (then 16 + 8 h .. + 7) of the lane's row
    const auto a = __builtin_amdgcn_permlane32_swap(w[p], w[2 + p], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[4 + p], w[6 + p], false, false);
    // across the 16s: rows 0 .. 15 in one, 16 .. 31 in the other
    const auto x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    lo[p] = x[0];
    lo[2 + p] = y[0];
    hi[p] = x[1];
    hi[2 + p] = y[1];
  }
}

// The first n (or all) of eight 16-bit elements to any address.
__device__ __forceinline__ void store_row8_bits(uint16_t* p, int n, u32x4_t v) {
  if (n >= 8) {
    ((Dwords4*)p)->v = v;
  } else if (n > 0) {
    if (n & 4) *(Dwords2*)p = Dwords2{{v[0], v[1]}};
    const uint32_t two = n & 4 ? v[2] : v[0], one = n & 2 ? (n & 4 ? v[3] : v[1]) : two;
    p += n & 4;
    if (n & 2) *(Dword*)p = Dword{two};
    if (n & 1) p[n & 2] = (uint16_t)one;
  }
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A matrix from one of its rows on, as a buffer resource: reads past its end give zeros.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ int buffer_size(long long bytes) {  // none where the row itself is past the end
  return (int)(uint32_t)min(max(bytes, 0ll), 0xfffffffell);
}
__device__ __forceinline__ i32x4_t buffer_from(const uint8_t* p, long long bytes) {
  const unsigned long long u = (unsigned long long)p;
  return {uniform((int)(uint32_t)u), uniform((int)((uint32_t)(u >> 32) & 0xffffu)),
          uniform(buffer_size(bytes)), 0x00020000};
}
// 16 bytes per lane from buffer + voff to LDS byte lds + 16 lane; as lds_dma16_asm, out of range lanes bring zeros.
__device__ __forceinline__ void buffer_dma16(i32x4_t buffer, uint32_t voff, uint32_t lds) {
  __asm__ volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(buffer),
                   "s"(lds)
                   : "memory");
}

// The same for loads that the compiler sees.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource_from(const uint8_t* p, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, uniform(buffer_size(bytes)), 0x00020000);
}

template <int N, class F>
__device__ __forceinline__ void unroll(F f) {  // f(0) .. f(N - 1) with constants
  if constexpr (N > 0) {
    unroll<N - 1>(f);
    f(std::integral_constant<int, N - 1>());
  }
}

// ---------------------------------------------------------------- ends of a tile
// A wave's 32 FM x 32 FN of c from row m0 and column n0 on.  Lane l + 32 h holds row l, columns 8 q + 4 h .. + 3 of each
// 32 x 32 piece; `bias` holds the wave's columns in LDS.
// To 16 bits: two rounds of lane swaps leave every lane with eight columns of one row and four lanes with 32.
template <int C, int ACT, int FM, int FN>
__device__ __forceinline__ void store_rows16(const GemmArgs& g, f32x16_t (&acc)[FM][FN], int m0, int n0, const float* bias) {
  int lane = threadIdx.x % kWave;
  __asm__ volatile("" : "+v"(lane));  // keeps addresses from being computed, and held, before the walk over the tiles
  const int row = lane % 16, col = (lane / 16 % 2) * 16 + (lane / 32) * 8;
  // rows past the last are past the buffer's end and not stored
  const __amdgpu_buffer_rsrc_t out =
      resource_from((const uint8_t*)g.c + (long long)m0 * g.n * 2, (long long)(g.m - m0) * g.n * 2);
  const bool inside = n0 + FN * 32 <= g.n && g.n % 2 == 0;  // uniform: whole pieces of eight columns, at 4-byte addresses
  uint32_t at = ((uint32_t)row * g.n + n0 + col) * 2;
  const uint32_t step = 16 * (uint32_t)g.n * 2;
  f32x4_t b[FN][4];
#pragma unroll
  for (int k = 0; k < FN; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) b[k][q] = *(const f32x4_t*)(bias + k * 32 + q * 8 + lane / 32 * 4);
  // A row's lines are written by neighbouring instructions: with the rows inside, as half lines a tile apart, the same
  // stores alone reach 3.4 TB/s instead of 4.9.
  unroll<FM>([&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    unroll<FN>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      f32x16_t c = acc[i][k];
#pragma unroll
      for (int r = 0; r < 16; ++r) c[r] += b[k][r / 4][r % 4];
      if (ACT == kActGeluTanh || (ACT == kActAny && g.act == kActGeluTanh))
#pragma unroll
        for (int r = 0; r < 16; ++r) c[r] = gelu_fast(c[r]);
      u32x4_t v[2];
      pack_rows<C>(c, v[0], v[1]);
      if (inside) {
        __builtin_amdgcn_raw_buffer_store_b128(v[0], out, at + k * 64, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(v[1], out, at + step + k * 64, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int m = m0 + i * 32 + j * 16 + row, n = n0 + k * 32 + col;
          if (m < g.m) store_row8_bits((uint16_t*)g.c + (long long)m * g.n + n, g.n - n, v[j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    at += 2 * step;
  });
}

// To fp32, four columns at a time: the result, or a share of the contracted dimension without bias and activation.
template <bool kShared, int FM, int FN>
__device__ __forceinline__ void store_rows32(const GemmArgs& g, f32x16_t (&acc)[FM][FN], int m0, int n0, int split,
                                             const float* bias) {
  int lane = threadIdx.x % kWave;
  __asm__ volatile("" : "+v"(lane));
  const int row = m0 + lane % 32, col = n0 + (lane / 32) * 4;
  float* base = kShared ? g.partial + (size_t)split * g.m * g.n : (float*)g.c;
  unroll<FM>([&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    const int m = row + i * 32;
    float* to = base + (size_t)m * g.n + col;
    unroll<FN * 4>([&](auto qc) __attribute__((always_inline)) {
      constexpr int q = decltype(qc)::value;
      const int n = g.n - col - q * 8;
      float c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = acc[i][q / 4][q % 4 * 4 + e];
      if (!kShared) {
        const f32x4_t b = *(const f32x4_t*)(bias + q * 8 + lane / 32 * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[e] += b[e];
          if (g.act == kActGeluTanh) c[e] = gelu_exact(c[e]);
        }
      }
      if (m < g.m) {
        if (n >= 4) {
          ((Dwords4*)(to + q * 8))->v = u32x4_t{__float_as_uint(c[0]), __float_as_uint(c[1]), __float_as_uint(c[2]),
                                                __float_as_uint(c[3])};
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (e < n) to[q * 8 + e] = c[e];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  });
}

// ---------------------------------------------------------------- the tile kernel
// A block of four waves (one per SIMD and tile quarter) computes tiles of kTile x kTile of c, 128 contracted positions
// (one scale block) at a time through two stages of LDS.  Stages are filled by LDS DMA with the 16-byte piece p of row r in
// place p ^ r ^ r / 8 (three bits of r, two of r / 8; swizzled at the source), so that 16 rows' reads of one piece are free
// of bank conflicts.  A wave keeps the operands of half a stage in registers and reads the other half's while its matrix
// instructions run; once the second half is read, the stage is free and takes the positions after next.  So one barrier
// per stage, behind which both the next stage's copies (issued a stage earlier) and this stage's reads are complete.
// Blocks stay, one per CU (kTile 256) or two (128), and walk over their items without a break in that sequence: the copies
// and reads for the next tile run while the last positions of a tile are multiplied.
// The matrix instruction's first operand is b and its second a: a lane then holds four consecutive columns of a row of c.
//
// What bounds it, kTile 256, per stage of 2048 matrix cycles (measured by stamps at 8192^3, 1.6 GHz under that load): 2130
// cycles; per tile 8500 for its end (adding, packing and storing 64K values) and 3000 for its start.  The LDS port moves a
// stage's 64 KB in and 128 KB out in about 1500 cycles; eight waves of 128 x 64 would read 192 KB and were 10% slower.
constexpr int kXcds = 8;
constexpr int gemm_blocks(int tile) { return tile == 256 ? 256 : 512; }

// The work of block `blockIdx.x`: every XCD (blocks are dealt to them in turn) takes a run of the items, its blocks take
// the run's items in turn.  An item is a tile and a share of the contracted dimension; tiles go down columns of kBand
// rows of tiles, so that the 32 blocks of an XCD share their operands in its L2.
struct GemmWalk {
  int first, last, step;  // items first, first + step, .. < last
};
__device__ __forceinline__ GemmWalk gemm_walk(int items, int blocks) {
  const int xcd = blockIdx.x % kXcds, slot = blockIdx.x / kXcds;
  const int share = items / kXcds, longer = items % kXcds, lo = xcd * share + min(xcd, longer);
  return {lo + slot, lo + share + (xcd < longer ? 1 : 0), blocks / kXcds};
}
struct GemmPlace {
  int m0, n0, k0, k1, split;
};
template <int BM, int BN, int kBand>
__device__ __forceinline__ GemmPlace gemm_place(const GemmArgs& g, int item) {
  const int mt = (g.m + BM - 1) / BM, nt = (g.n + BN - 1) / BN;
  const int tile = item / g.splits, split = item - tile * g.splits;
  const int band = tile / (kBand * nt), rows = min(kBand, mt - band * kBand), in = tile - band * kBand * nt;
  const int n = in / rows, m = band * kBand + in - n * rows;
  const int share = g.kb / g.splits, longer = g.kb - share * g.splits;  // the first `longer` shares have one more
  const int k0 = split * share + min(split, longer);
  return {uniform(m * BM), uniform(n * BN), uniform(k0), uniform(k0 + share + (split < longer ? 1 : 0)), uniform(split)};
}

// A: the 8-bit type of a.  C: the type of c, or kShare.  ACT: the activation, or kActAny to ask the arguments.
// c in fp32 multiplies in bf16 (above), with the scales taken in as the operands widen.
template <int A, int C, int ACT, int kTile>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kTile == 256 ? 1 : 2, kTile == 256 ? 1 : 2)))
fp8_gemm_tile_kernel(GemmArgs g) {
  constexpr bool kWide = C == kRowF32 || C == kShareWide, kShared = C == kShare || C == kShareWide;
  constexpr int kWaves = 4, kPart = kTile / 2, F = kPart / 32;  // the wave's part of the tile, in rows and in 32s of rows
  constexpr int kStageBytes = 2 * kTile * 128;
  constexpr int kCopies = kTile / 8 / kWaves;  // 1 KB copies per wave, stage and operand
  constexpr int kBand = 8;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStageBytes];
  __shared__ __attribute__((aligned(16))) float bias_part[kWaves][kPart];
  const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
  const int l = lane % 32, h = lane / 32;
  const int wm = (wave / 2) * kPart, wn = (wave % 2) * kPart;
  const int mt = (g.m + kTile - 1) / kTile, nt = (g.n + kTile - 1) / kTile;
  const GemmWalk walk = gemm_walk(mt * nt * g.splits, gemm_blocks(kTile));
  if (walk.first >= walk.last) return;
  auto place = [&](int item) __attribute__((always_inline)) { return gemm_place<kTile, kTile, kBand>(g, item); };

  // The copies: lane i of a copy writes piece i % 8 of row i / 8 of its eight rows.  They run two stages ahead of the
  // multiplication, into the next item, or the last one again once there is no other.
  const uint32_t a_row = (uint32_t)g.a_row, b_row = (uint32_t)g.b_row;
  const uint32_t piece = ((lane % 8) ^ (lane / 8) ^ (wave & 3)) * 16;
  const uint32_t va = (wave * 8 + lane / 8) * a_row + piece, vb = (wave * 8 + lane / 8) * b_row + piece;
  const uint32_t lds0 = lds_addr(lds) + wave * 1024;
  i32x4_t buf_a, buf_b;
  uint32_t c_k, c_dst = lds0;
  auto copy_from = [&](const GemmPlace& p) __attribute__((always_inline)) {
    buf_a = buffer_from(g.a + (long long)p.m0 * g.a_row, (g.m - 1 - p.m0) * g.a_row + g.kb * 128);
    buf_b = buffer_from(g.b + (long long)p.n0 * g.b_row, (g.n - 1 - p.n0) * g.b_row + g.kb * 128);
    c_k = p.k0 * 128;
  };
  auto copy = [&](int i) __attribute__((always_inline)) {  // the i-th of a stage's 2 kCopies
    if (i < kCopies) buffer_dma16(buf_a, va + (i * kWaves * 8 * a_row + c_k), c_dst + i * kWaves * 1024);
    else buffer_dma16(buf_b, vb + ((i - kCopies) * kWaves * 8 * b_row + c_k), c_dst + kTile * 128 + (i - kCopies) * kWaves * 1024);
  };
  // A stage's last kLate copies are left to the first half of the next stage.
  constexpr int kLate = kCopies / 2;
  i32x4_t late_b;
  uint32_t late_k, late_dst;
  auto copy_late = [&](int i) __attribute__((always_inline)) {
    buffer_dma16(late_b, vb + ((i - kCopies) * kWaves * 8 * b_row + late_k), late_dst + kTile * 128 + (i - kCopies) * kWaves * 1024);
  };
  auto copy_next = [&]() __attribute__((always_inline)) {
    late_b = buf_b;
    late_k = c_k;
    late_dst = c_dst;
    c_k += 128;
    c_dst = lds0 + (c_dst == lds0 ? kStageBytes : 0);
    if (g.kb == 1) buf_a[2] = buf_b[2] = 0;  // an item has two stages at least: one of zeros
  };

  // The scales of the wave's rows, a byte of sa and sb each; past the last row the buffer gives zeros.  Loaded two stages
  // ahead and taken behind a stage's barrier: the compiler's wait for them then finds nothing outstanding, where one
  // behind the copies, which it does not count, would wait for those too.
  const uint32_t vsa = l * (uint32_t)g.a_scale_row, vsb = g.b_shift ? 0 : l * (uint32_t)g.b_scale_row;
  __amdgpu_buffer_rsrc_t buf_sa, buf_sb;
  int s_k;
  int na[F], nb[F], sa, sb, sa1, sb1;
  auto scales_from = [&](const GemmPlace& p) __attribute__((always_inline)) {
    const int b0 = p.n0 >> g.b_shift, b_last = (g.n - 1) >> g.b_shift;
    buf_sa = resource_from(g.a_scale + (long long)p.m0 * g.a_scale_row,
                           (g.m - 1 - p.m0) * g.a_scale_row + (g.kb - 1) * g.a_scale_col + 1);
    buf_sb = resource_from(g.b_scale + (long long)b0 * g.b_scale_row,
                           (b_last - b0) * g.b_scale_row + (g.kb - 1) * g.b_scale_col + 1);
    s_k = p.k0;
  };
  auto load_scale = [&](int& to, __amdgpu_buffer_rsrc_t buf, uint32_t voff, int row, long long row_stride,
                        long long col_stride) __attribute__((always_inline)) {
    const uint32_t past = s_k < g.kb ? 0 : 0x80000000u;  // of the stage of zeros: past any buffer's end
    to = __builtin_amdgcn_raw_buffer_load_b8(buf, voff + (row * (uint32_t)row_stride + s_k * (uint32_t)col_stride + past), 0, 0);
  };
  auto load_scale_a = [&](int i) __attribute__((always_inline)) {
    load_scale(na[i], buf_sa, vsa, wm + i * 32, g.a_scale_row, g.a_scale_col);
  };
  auto load_scale_b = [&](int i) __attribute__((always_inline)) {
    load_scale(nb[i], buf_sb, vsb, (wn + i * 32) >> g.b_shift, g.b_scale_row, g.b_scale_col);
  };

  // The bias: a lane loads that of a column or two of the wave's, an item ahead and in both widths, without a branch (at
  // whose end a wait would be for the last item's stores as well); it stays in LDS until the end of the item.
  constexpr int kBias = (kPart + kWave - 1) / kWave;
  int raw[2 * kBias];
  const __amdgpu_buffer_rsrc_t buf_bias = resource_from(
      (const uint8_t*)g.bias, kShared || g.bias == nullptr ? 0 : (long long)g.n * (g.bias_type == kRowF32 ? 4 : 2));
  auto load_bias = [&](const GemmPlace& p) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBias; ++i) {
      const int n = p.n0 + wn + i * kWave + lane;
      raw[i] = __builtin_amdgcn_raw_buffer_load_b32(buf_bias, n * 4, 0, 0);
      raw[kBias + i] = __builtin_amdgcn_raw_buffer_load_b16(buf_bias, n * 2, 0, 0);
    }
  };
  auto spread_bias = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kBias; ++i) {
      const uint16_t half = (uint16_t)raw[kBias + i];
      const float wide = g.bias_type == kRowBf16 ? bf16_to_f32(half) : (float)__builtin_bit_cast(_Float16, half);
      if (i * kWave + lane < kPart)
        bias_part[wave][i * kWave + lane] = g.bias_type == kRowF32 ? __int_as_float(raw[i]) : wide;
    }
  };

  auto take_scales = [&]() __attribute__((always_inline)) {
    sa1 = na[0];
    sb1 = nb[0];
#pragma unroll
    for (int i = 1; i < F; ++i) {
      sa1 |= na[i] << (8 * i);
      sb1 |= nb[i] << (8 * i);
    }
    __asm__ volatile("" : "+v"(sa1), "+v"(sb1));
#pragma unroll
    for (int i = 0; i < 2 * kBias; ++i) __asm__ volatile("" : "+v"(raw[i]));
  };

  int off[2][2];  // of a row's pieces 4 j + 2 h and 4 j + 2 h + 1
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) off[j][e] = l * 128 + (((4 * j + 2 * h + e) ^ ((l ^ (l >> 3)) & 7)) << 4);
  f32x16_t acc[F][F];
  i32x8_t f[2][2 * F];  // operands of b, then of a, of the two halves of a stage
  // Half e of operand r: of the 32 rows of b or a that it holds.
  auto read = [&](int stage, auto jc, auto rc, auto ec) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value, r = decltype(rc)::value, e = decltype(ec)::value;
    const int rows = r < F ? kTile + wn + r * 32 : wm + (r - F) * 32;
    const u32x4_t x = *(const u32x4_t*)(lds + stage + rows * 128 + off[j][e]);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[j][r][4 * e + i] = (int)x[i];
  };
  // Half a stage on the operands in registers.  Those of the other half (of stage `next`) are read between its
  // instructions, one read (four waves' take 32 of an instruction's 64 cycles on the LDS port) and in the second half one
  // copy (16 cycles of the memory pipe each) at a time: in bursts the queues fill, and the wave waits to issue with its
  // matrix unit idle.
  auto half_stage = [&](auto half, int next) __attribute__((always_inline)) {
    constexpr int j = decltype(half)::value, kReads = 4 * F, kSlots = F * F;
    u32x4_t wide_b[kWide ? F : 1][4];
    if constexpr (kWide) unroll<F>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      widen<kFp8E4m3>(f[j][k], (sb >> (8 * k)) & 0xff, wide_b[k]);
    });
    unroll<kSlots>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = decltype(tc)::value, i = t / F, k = t % F;
      if constexpr (kWide) {
        u32x4_t wide_a[4];
        widen<A>(f[j][F + i], (sa >> (8 * i)) & 0xff, wide_a);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][k] = mfma32x32x16(as_bf16x8(wide_b[k][e]), as_bf16x8(wide_a[e]), acc[i][k]);
      } else {
        acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f[j][k], f[j][F + i], acc[i][k], 0, A, k, sb, i, sa);
      }
      constexpr int read_slots = kSlots > 8 ? kSlots - 2 : kSlots;
      constexpr int r0 = t * kReads / read_slots, r1 = (t + 1) * kReads / read_slots;
      unroll<r1 - r0>([&](auto rc) __attribute__((always_inline)) {
        constexpr int r = r0 + decltype(rc)::value;
        if constexpr (r < kReads)
          read(next, std::integral_constant<int, j ^ 1>(), std::integral_constant<int, r / 2>(),
               std::integral_constant<int, r % 2>());
      });
      if constexpr (j == 0 && t < kLate) copy_late(2 * kCopies - kLate + t);
      if constexpr (j == 1) {
        if constexpr (t == 0) take_scales();
        constexpr int now = 2 * kCopies - kLate, c0 = t * now / kSlots, c1 = (t + 1) * now / kSlots;
        unroll<c1 - c0>([&](auto cc) __attribute__((always_inline)) { copy(c0 + decltype(cc)::value); });
        if constexpr (t >= kSlots - F) {
          load_scale_a(t - (kSlots - F));
          load_scale_b(t - (kSlots - F));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  const std::integral_constant<int, 0> first;
  const std::integral_constant<int, 1> second;
  auto hold_sums = [&]() __attribute__((always_inline)) {  // in the accumulation registers
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int k = 0; k < F; ++k) __asm__ volatile("" : "+a"(acc[i][k]));
  };

  GemmPlace p = place(walk.first);
  copy_from(p);
  scales_from(p);
  load_bias(p);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      load_scale_a(i);
      load_scale_b(i);
    }
    ++s_k;
    if (s == 0) {
      take_scales();
      sa = sa1;
      sb = sb1;
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * kCopies; ++i) copy(i);
  copy_next();
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2 * kCopies - kLate; ++i) copy(i);
  copy_next();
  unroll<4 * F>([&](auto rc) __attribute__((always_inline)) {
    constexpr int r = decltype(rc)::value;
    read(0, first, std::integral_constant<int, r / 2>(), std::integral_constant<int, r % 2>());
  });

  int stage = 0;
  for (int item = walk.first; item < walk.last; item += walk.step) {
    const GemmPlace next = place(item + walk.step < walk.last ? item + walk.step : item);
    spread_bias();
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int k = 0; k < F; ++k) acc[i][k] = f32x16_t{};
    hold_sums();
#pragma unroll 1
    for (int left = max(p.k1 - p.k0, 2); left > 0; --left) {
      if (left == 2) {  // here, not where they are used: a branch between the halves would let instructions sink past it
        scales_from(next);
        copy_from(next);
      }
      half_stage(first, stage);
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      stage ^= kStageBytes;
      half_stage(second, stage);
      ++s_k;
      copy_next();
      sa = sa1;
      sb = sb1;
    }
    hold_sums();
    load_bias(next);
    const int m0 = p.m0 + wm, n0 = p.n0 + wn;
    if constexpr (kShared || C == kRowF32) {
      store_rows32<kShared>(g, acc, m0, n0, p.split, bias_part[wave]);
    } else {
      store_rows16<C, ACT>(g, acc, m0, n0, bias_part[wave]);
    }
    p = next;
  }
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may land in LDS that is another block's by then
}

// Launches of the instances, each compiled in one of the fp8_gemm_*.hip files.
void launch_gemm_256(const GemmArgs& g, int a_type, int c, hipStream_t s);        // c: a 16-bit type or kShare
void launch_gemm_256_e5m2(const GemmArgs& g, int c, hipStream_t s);
void launch_gemm_128(const GemmArgs& g, int a_type, int c, hipStream_t s);        // any c

}  // namespace svoo
