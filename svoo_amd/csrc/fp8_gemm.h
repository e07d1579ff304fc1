// Product of 8-bit matrices with a power-of-two scale per block of 128 along the contracted dimension:
//   c[m][n] = act(sum_k 2^(ea[m][k/128]) a[m][k] 2^(eb[n or n/128][k/128]) b[n][k] + bias[n])
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies the scales in and accumulates in fp32.  A lane's 32 bytes of an operand
// may be any 32 of the 128 contracted positions as long as both operands agree, and one scale covers all of them.
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
// before they go to the fp32 accumulator (measured with powers of two; the same for the unscaled instructions): 1.5e-5 to
// 3.5e-5 of a random sum's size, at most a sixth of the rounding to fp16 and a fiftieth of that to bf16.  A caller who asks
// for fp32 gets sums in fp32: the values widen to bf16, scale included, and go through the bf16 instructions, which round
// nothing else, at half the rate (4096 x 5120 x 5120 197 us, 1.1 PFLOP/s).  Widening is exact for all values of e4m3 with
// scales of 2^-124 to 2^119, of e5m2 with 2^-117 to 2^112; past those, values below 2^-126 are rounded to steps of 2^-133
// and values from 2^128 on become infinite.
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

// Two neighbouring 16 x 16 pieces as 16 bits each: lane 16 b + 32 h + i gets columns 16 b + 8 h .. + 7 of row i.
template <int T>
__device__ __forceinline__ u32x4_t pack_rows(f32x4_t left, f32x4_t right) {
  uint32_t w[2][2];  // columns 4 (lane / 16) + 2 p and the next
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const f32x4_t c = k ? right : left;
      w[k][p] = T == kRowBf16 ? cvt_pk_bf16(c[2 * p], c[2 * p + 1])
                              : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)c[2 * p]) |
                                    ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)c[2 * p + 1]) << 16);
    }
  u32x4_t v;
#pragma unroll
  for (int p = 0; p < 2; ++p) {  // columns 4 .. 7 of each eight from the lanes 16 on
    const auto x = __builtin_amdgcn_permlane16_swap(w[0][p], w[1][p], false, false);
    v[p] = x[0];
    v[2 + p] = x[1];
  }
  return v;
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
// 16 bytes per lane from buffer + soff + voff to LDS byte lds + kAt + 16 lane.  Lanes out of range bring zeros: here rows
// past the last, whose voff alone is past the end.
template <int kAt>
__device__ __forceinline__ void buffer_dma16(i32x4_t buffer, uint32_t voff, uint32_t soff, uint32_t lds) {
  __asm__ volatile("s_add_u32 m0, %2, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds" ::"v"(voff), "s"(buffer),
                   "s"(lds), "s"(soff), "i"(kAt)
                   : "memory", "m0", "scc");
}
// An element of 1, 2 or 4 bytes per lane to words of LDS.
template <int kBytes, int kAt>
__device__ __forceinline__ void buffer_dma_words(i32x4_t buffer, uint32_t voff, uint32_t lds) {
  if constexpr (kBytes == 1)
    __asm__ volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_ubyte %0, %1, 0 offen lds" ::"v"(voff), "s"(buffer),
                     "s"(lds), "i"(kAt)
                     : "memory", "m0", "scc");
  else if constexpr (kBytes == 2)
    __asm__ volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_ushort %0, %1, 0 offen lds" ::"v"(voff), "s"(buffer),
                     "s"(lds), "i"(kAt)
                     : "memory", "m0", "scc");
  else
    __asm__ volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(buffer),
                     "s"(lds), "i"(kAt)
                     : "memory", "m0", "scc");
}
template <class T>
__device__ __forceinline__ const __attribute__((address_space(3))) T* lds_at(uint32_t at) {
  return (const __attribute__((address_space(3))) T*)(uintptr_t)at;
}
// Until no more than N of the wave's loads and stores are outstanding, in a form that the compiler counts.
template <int N>
__device__ __forceinline__ void wait_vmem() {
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4 << 14));
  __asm__ volatile("" ::: "memory");
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
// A wave's 16 FM x 16 FN of c from row m0 and column n0 on.  Lane l + 16 g holds row l, columns 4 g .. + 3 of each
// 16 x 16 piece, and the bias of columns l + 16 g and, of 128, + 64 in `bias`.
template <int FN>
__device__ __forceinline__ f32x4_t bias_of(const float (&bias)[(FN * 16 + kWave - 1) / kWave], int k, int lane) {
  f32x4_t b;
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = __shfl(bias[k / 4], k % 4 * 16 + lane / 16 * 4 + e);
  return b;
}
// To 16 bits: a lane swap between two pieces leaves every lane with eight columns of one row and four lanes with 32.
template <int C, int ACT, int FM, int FN>
__device__ __forceinline__ void store_rows16(const GemmArgs& g, f32x4_t (&acc)[FM][FN], int m0, int n0,
                                             const float (&bias)[(FN * 16 + kWave - 1) / kWave]) {
  int lane = threadIdx.x % kWave;
  __asm__ volatile("" : "+v"(lane));  // keeps addresses from being computed, and held, before the walk over the tiles
  const int row = lane % 16, col = (lane / 16 % 2) * 16 + (lane / 32) * 8;
  // rows past the last are past the buffer's end and not stored
  const __amdgpu_buffer_rsrc_t out =
      resource_from((const uint8_t*)g.c + (long long)m0 * g.n * 2, (long long)(g.m - m0) * g.n * 2);
  const bool inside = n0 + FN * 16 <= g.n && g.n % 2 == 0;  // uniform: whole pieces of eight columns, at 4-byte addresses
  uint32_t at = ((uint32_t)row * g.n + n0 + col) * 2;
  const uint32_t step = 16 * (uint32_t)g.n * 2;
  f32x4_t b[FN];
#pragma unroll
  for (int k = 0; k < FN; ++k) b[k] = bias_of<FN>(bias, k, lane);
  // A row's lines are written by neighbouring instructions: with the rows inside, as half lines a tile apart, the same
  // stores alone reach 3.4 TB/s instead of 4.9.
  unroll<FM>([&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    unroll<FN / 2>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      f32x4_t c[2] = {acc[i][2 * k], acc[i][2 * k + 1]};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          c[h][r] += b[2 * k + h][r];
          if (ACT == kActGeluTanh || (ACT == kActAny && g.act == kActGeluTanh)) c[h][r] = gelu_fast(c[h][r]);
        }
      const u32x4_t v = pack_rows<C>(c[0], c[1]);
      if (inside) {
        __builtin_amdgcn_raw_buffer_store_b128(v, out, at + k * 64, 0, 0);
      } else {
        const int m = m0 + i * 16 + row, n = n0 + k * 32 + col;
        if (m < g.m) store_row8_bits((uint16_t*)g.c + (long long)m * g.n + n, g.n - n, v);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    at += step;
  });
}

// To fp32, four columns at a time: the result, or a share of the contracted dimension without bias and activation.
template <bool kShared, int FM, int FN>
__device__ __forceinline__ void store_rows32(const GemmArgs& g, f32x4_t (&acc)[FM][FN], int m0, int n0, int split,
                                             const float (&bias)[(FN * 16 + kWave - 1) / kWave]) {
  int lane = threadIdx.x % kWave;
  __asm__ volatile("" : "+v"(lane));
  const int row = m0 + lane % 16, col = n0 + (lane / 16) * 4;
  float* base = kShared ? g.partial + (size_t)split * g.m * g.n : (float*)g.c;
  unroll<FM>([&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    const int m = row + i * 16;
    float* to = base + (size_t)m * g.n + col;
    unroll<FN>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      const int n = g.n - col - k * 16;
      f32x4_t c = acc[i][k];
      if (!kShared) {
        const f32x4_t b = bias_of<FN>(bias, k, lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[e] += b[e];
          if (g.act == kActGeluTanh) c[e] = gelu_exact(c[e]);
        }
      }
      if (m < g.m) {
        if (n >= 4) {
          ((Dwords4*)(to + k * 16))->v = u32x4_t{__float_as_uint(c[0]), __float_as_uint(c[1]), __float_as_uint(c[2]),
                                                 __float_as_uint(c[3])};
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (e < n) to[k * 16 + e] = c[e];
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
// of bank conflicts.  A wave holds one stage's operands in registers and reads the next ones while its matrix instructions
// run.  A barrier in the middle of a stage and one at its end each free half of a stage's place, which the copies for the
// same half of the stage after next then fill: they have a stage's time to land, and go out evenly.  (With one barrier
// they had half of it, in bursts that kept the waves waiting to issue: 3000 cycles a stage instead of 2500.)
// Blocks stay, one per CU (kTile 256) or two (128), and walk over their items without a break in that sequence: the copies
// and reads for the next tile run while the last positions of a tile are multiplied.
// The matrix instruction's first operand is b and its second a: a lane then holds four consecutive columns of a row of c.
// The 16 x 16 x 128 form sustains 4.25 PFLOP/s from registers on random values, the 32 x 32 x 64 form 3.95: the clock
// falls with the power that they take.
//
// What bounds it, kTile 256 (measured by stamps): per stage of 2048 matrix cycles 2500, 290 of them lost to barriers and to
// instructions that wait for each other's issue, the rest to copies; per tile 9500 to add, pack and store 64K values, and
// behind them the stores themselves (all blocks end a tile together), which at 1536 contracted positions take a third of
// the time.  The clock is 1.8 GHz under random values and 2.3 under zeros.  8192^3 380 us (2.9 PFLOP/s),
// 32760 x 1536 x 8960 330 us (2.7), 32760 x 8960 x 1536 415 us (2.2, 1.4 TB/s of stores), 8960 x 1536 x 32768 350 us (2.6).
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
  constexpr int kWaves = 4, kPart = kTile / 2, F = kPart / 16;  // the wave's part of the tile, in rows and in 16s of rows
  constexpr int kStageBytes = 2 * kTile * 128;
  constexpr int kCopies = kTile / 8 / kWaves;  // 1 KB copies per wave, stage and operand
  constexpr int kScaleBytes = 2 * kTile * 4, kScaleCopies = kTile / 128;  // a word per row of a and b and stage
  // 4, 5, 6, 8, 11 and 16 rows of 256: 391, 397, 400, 406, 415 and 420 us at 32760 x 1536 x 8960, within 2% elsewhere
  constexpr int kBand = kTile == 256 ? 4 : 8;
  constexpr int kBiasAt = 2 * kStageBytes + 2 * kScaleBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBiasAt + kWaves * kPart * 4];
  const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
  const int wm = (wave / 2) * kPart, wn = (wave % 2) * kPart;
  const int mt = (g.m + kTile - 1) / kTile, nt = (g.n + kTile - 1) / kTile;
  const GemmWalk walk = gemm_walk(mt * nt * g.splits, gemm_blocks(kTile));
  if (walk.first >= walk.last) return;
  auto place = [&](int item) __attribute__((always_inline)) { return gemm_place<kTile, kTile, kBand>(g, item); };

  // The copies: lane i of a copy writes piece i % 8 of row i / 8 of its eight rows, or the scale of row i of 64.  They run
  // two stages ahead of the multiplication, into the next item, or the last one again once there is no other.
  const uint32_t piece = ((lane % 8) ^ (lane / 8) ^ (wave & 3)) * 16;
  uint32_t va[kCopies], vb[kCopies], vs[kScaleCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    va[i] = ((i * kWaves + wave) * 8 + lane / 8) * (uint32_t)g.a_row + piece;
    vb[i] = ((i * kWaves + wave) * 8 + lane / 8) * (uint32_t)g.b_row + piece;
  }
  auto scale_of_b = [&](int i) __attribute__((always_inline)) { return (wave + i * kWaves) * kWave >= kTile; };
  uint32_t s_step[kScaleCopies];
#pragma unroll
  for (int i = 0; i < kScaleCopies; ++i) {
    const int row = (wave + i * kWaves) * kWave % kTile + lane;
    const bool of_b = scale_of_b(i);
    vs[i] = (of_b ? row >> g.b_shift : row) * (uint32_t)(of_b ? g.b_scale_row : g.a_scale_row);
    s_step[i] = g.kb == 1 ? 0 : (uint32_t)(of_b ? g.b_scale_col : g.a_scale_col);
  }
  const uint32_t lds0 = lds_addr(lds) + wave * 1024, lds_s0 = lds_addr(lds) + 2 * kStageBytes + wave * kWave * 4;
  const uint32_t k_step = g.kb == 1 ? 0 : 128;
  i32x4_t buf_a, buf_b, buf_s[kScaleCopies];
  uint32_t c_k, s_k[kScaleCopies], c_dst = lds0, s_dst = lds_s0;
  struct Source {
    i32x4_t a, b, s[kScaleCopies];
    uint32_t k, s_k[kScaleCopies];
  };
  auto source = [&](const GemmPlace& p) __attribute__((always_inline)) {
    Source s;
    s.a = buffer_from(g.a + (long long)p.m0 * g.a_row, (g.m - 1 - p.m0) * g.a_row + g.kb * 128);
    s.b = buffer_from(g.b + (long long)p.n0 * g.b_row, (g.n - 1 - p.n0) * g.b_row + g.kb * 128);
    s.k = p.k0 * 128;
#pragma unroll
    for (int i = 0; i < kScaleCopies; ++i) {
      const int b0 = p.n0 >> g.b_shift, b_last = (g.n - 1) >> g.b_shift;
      s.s[i] = scale_of_b(i) ? buffer_from(g.b_scale + (long long)b0 * g.b_scale_row,
                                           (b_last - b0) * g.b_scale_row + (g.kb - 1) * g.b_scale_col + 1)
                             : buffer_from(g.a_scale + (long long)p.m0 * g.a_scale_row,
                                           (g.m - 1 - p.m0) * g.a_scale_row + (g.kb - 1) * g.a_scale_col + 1);
      s.s_k[i] = p.k0 * s_step[i];
    }
    return s;
  };
  auto copy_from = [&](const Source& s) __attribute__((always_inline)) {
    buf_a = s.a;
    buf_b = s.b;
    c_k = s.k;
#pragma unroll
    for (int i = 0; i < kScaleCopies; ++i) {
      buf_s[i] = s.s[i];
      s_k[i] = s.s_k[i];
    }
  };
  auto copy_zeros = [&]() __attribute__((always_inline)) {  // out of buffers without a byte
    buf_a[2] = buf_b[2] = 0;
#pragma unroll
    for (int i = 0; i < kScaleCopies; ++i) buf_s[i][2] = 0;
  };
  // A stage's copies, in two halves: first the scales and, of a and b, the first half of each wave's rows.
  auto copy_rows = [&](auto half, auto ic) __attribute__((always_inline)) {  // the i-th of kCopies
    constexpr int n = kCopies / 2, q = decltype(ic)::value % n, i = q / (n / 2) * n + decltype(half)::value * (n / 2) + q % (n / 2);
    if constexpr (decltype(ic)::value < n) buffer_dma16<i * kWaves * 1024>(buf_a, va[i], c_k, c_dst);
    else buffer_dma16<kTile * 128 + i * kWaves * 1024>(buf_b, vb[i], c_k, c_dst);
  };
  auto copy_scales = [&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    buffer_dma_words<1, i * kWaves * kWave * 4>(buf_s[i], vs[i] + s_k[i], s_dst);
  };
  constexpr int kFirst = kCopies + kScaleCopies;
  auto copy_first = [&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < kScaleCopies) copy_scales(ic);
    else copy_rows(std::integral_constant<int, 0>(), std::integral_constant<int, i - kScaleCopies>());
  };
  auto copy_second = [&](auto ic) __attribute__((always_inline)) { copy_rows(std::integral_constant<int, 1>(), ic); };
  auto copy_next = [&]() __attribute__((always_inline)) {
    c_k += k_step;
    c_dst = 2 * lds0 + kStageBytes - c_dst;
    s_dst = 2 * lds_s0 + kScaleBytes - s_dst;
#pragma unroll
    for (int i = 0; i < kScaleCopies; ++i) s_k[i] += s_step[i];
  };

  // The scales of the wave's rows: lane l reads that of row l of each 64 and gets those of rows l % 16, + 16, + 32 and + 48
  // as the bytes of a word.
  constexpr int kScales = kPart / kWave;
  int na[kScales], nb[kScales], sa[kScales], sb[kScales], sa1[kScales], sb1[kScales];
  uint32_t s_at = lds_addr(lds) + 2 * kStageBytes + lane * 4, s_turn = kScaleBytes;
  auto read_scale = [&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < kScales) na[i] = *lds_at<int>(s_at + (wm + i * kWave) * 4);
    else nb[i - kScales] = *lds_at<int>(s_at + (kTile + wn + (i - kScales) * kWave) * 4);
  };
  auto word = [&](int v) __attribute__((always_inline)) {
    const auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // rows of 16 lanes 0 0 2 2, 1 1 3 3
    const int t = x[0] | x[1] << 8;
    const auto y = __builtin_amdgcn_permlane32_swap(t, t, false, false);
    return (int)(y[0] | y[1] << 16);
  };
  auto take_scale = [&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i < kScales) sa1[i] = word(na[i]);
    else sb1[i - kScales] = word(nb[i - kScales]);
  };

  // The bias of the wave's columns, copied at an item's start and read at its end, when it has landed long since (there are
  // two stages at least).
  const i32x4_t buf_bias =
      buffer_from((const uint8_t*)g.bias, kShared || g.bias == nullptr ? 0 : (long long)g.n * (g.bias_type == kRowF32 ? 4 : 2));
  const uint32_t bias_at = lds_addr(lds) + kBiasAt + wave * kPart * 4;
  auto copy_bias = [&](int n0) __attribute__((always_inline)) {
    if (g.bias_type == kRowF32) unroll<kScales>([&](auto ic) __attribute__((always_inline)) {
      buffer_dma_words<4, decltype(ic)::value * kWave * 4>(buf_bias, (n0 + decltype(ic)::value * kWave + lane) * 4, bias_at);
    });
    else unroll<kScales>([&](auto ic) __attribute__((always_inline)) {
      buffer_dma_words<2, decltype(ic)::value * kWave * 4>(buf_bias, (n0 + decltype(ic)::value * kWave + lane) * 2, bias_at);
    });
  };
  auto read_bias = [&](float (&bias)[kScales]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
      const int raw = *lds_at<int>(bias_at + (i * kWave + lane) * 4);
      const float wide = g.bias_type == kRowBf16 ? bf16_to_f32((uint16_t)raw) : (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
      bias[i] = g.bias_type == kRowF32 ? __int_as_float(raw) : wide;
    }
  };

  // LDS bytes of pieces 2 g and 2 g + 1 of row l of the wave's part of b and a, in 16 rows from a multiple of 32 on and in
  // the next; of the stage that is read.
  uint32_t off[2][2][2];
  const int l = lane % 16, lg = lane / 16;
#pragma unroll
  for (int o = 0; o < 2; ++o)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        off[o][j][e] = lds_addr(lds) + ((o ? wm : kTile + wn) + l) * 128 + (((2 * lg + e) ^ ((l ^ (l >> 3) ^ (2 * j)) & 7)) << 4);
  uint32_t stage_turn = kStageBytes;  // to the other stage
  auto read_from_next = [&](int o) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) off[o][j][e] += stage_turn;
  };
  f32x4_t acc[F][F];
  i32x8_t f[2 * F], spare;  // operands of b, then of a, of 16 rows each
  // Half e of operand r, or of one of the next stage's that waits for its registers.
  auto read = [&](auto rc, auto ec, i32x8_t& to) __attribute__((always_inline)) {
    constexpr int r = decltype(rc)::value, e = decltype(ec)::value;
    const u32x4_t x = *lds_at<u32x4_t>(off[r / F][r % 2][e] + r % F * 2048);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[4 * e + i] = (int)x[i];
  };
  auto read_part = [&](auto first, auto qc) __attribute__((always_inline)) {  // the q-th of operands `first` on
    constexpr int r = decltype(first)::value + decltype(qc)::value / 2;
    read(std::integral_constant<int, r>(), std::integral_constant<int, decltype(qc)::value % 2>(), f[r]);
  };
  // Half a stage: the first or second half of the wave's rows with all its columns, in quarters: rows 0 with columns 0 and
  // 1, rows 1 with columns 1 and 0.  So a quarter leaves the registers of one half operand free and the next but one needs
  // another: columns 1, rows 1, then from the next stage rows 0 and (each as soon as it is used for the last time, the
  // last through spare registers) columns 0.  Reads, copies (16 cycles of the memory pipe each) and what else there is go
  // one at a time between the instructions: while the wave waits to issue one, its matrix unit idles.
  auto half_stage = [&](auto half) __attribute__((always_inline)) {
    constexpr int j = decltype(half)::value, H = F / 2, kSlots = F * H;
    u32x4_t wide_a[kWide ? H : 1][4], wide_b[4];
    if constexpr (kWide) unroll<H>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = j * H + decltype(ic)::value;
      widen<A>(f[F + i], (sa[i / 4] >> (8 * (i % 4))) & 0xff, wide_a[decltype(ic)::value]);
    });
    unroll<kSlots>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = decltype(tc)::value, quarter = t / (H * H), u = t % (H * H), in = u % H, kk = u / H;
      constexpr int i = j * H + in, k = (quarter ^ j) * H + kk;
      if constexpr (kWide) {
        if constexpr (in == 0) widen<kFp8E4m3>(f[k], (sb[k / 4] >> (8 * (k % 4))) & 0xff, wide_b);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(wide_b[e]), as_bf16x8(wide_a[in][e]), acc[i][k], 0, 0, 0);
      } else {
        acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(f[k], f[F + i], acc[i][k], 0, A, k % 4, sb[k / 4], i % 4,
                                                                     sa[i / 4]);
      }
      // q0 .. q1 - 1: the reads of a quarter's half operand that go behind this instruction
      constexpr int span = H == 2 ? 4 : j == 0 ? 12 : 16;
      constexpr int q0 = (u * F + span - 1) / span, q1 = std::min(((u + 1) * F + span - 1) / span, F);
      constexpr int from = j == 1 ? F : quarter == 0 ? H : F + H;
      if constexpr (j == 0 || quarter == 0) {
        unroll<std::max(q1 - q0, 0)>([&](auto qc) __attribute__((always_inline)) {
          read_part(std::integral_constant<int, from>(), std::integral_constant<int, q0 + decltype(qc)::value>());
        });
      } else if constexpr (in < 2) {
        if constexpr (kk == 0) read(std::integral_constant<int, H - 1>(), std::integral_constant<int, in>(), spare);
        else read_part(std::integral_constant<int, kk - 1>(), std::integral_constant<int, in>());
      }
      constexpr int n = j == 0 ? kFirst : kCopies, c0 = t * n / kSlots, c1 = (t + 1) * n / kSlots;
      unroll<c1 - c0>([&](auto cc) __attribute__((always_inline)) {
        constexpr std::integral_constant<int, c0 + decltype(cc)::value> c;
        if constexpr (j == 0) copy_first(c);
        else copy_second(c);
      });
      if constexpr (j == 0) {
        constexpr int moves = 16 / F;  // before the spare operand's turn
        if constexpr (t * moves < 8) {
#pragma unroll
          for (int e = 0; e < moves; ++e) f[H - 1][t * moves + e] = spare[t * moves + e];
        }
        if constexpr (t == H * H) read_from_next(0);
        if constexpr (t == kSlots - 1) {
          read_from_next(1);
          stage_turn = -stage_turn;
        }
      } else {
        constexpr int every = kSlots / (4 * kScales);  // scales: all reads, then all words
        if constexpr (t % every == every / 2) {
          constexpr int x = t / every;
          if constexpr (x < 2 * kScales) read_scale(std::integral_constant<int, x>());
          else take_scale(std::integral_constant<int, x - 2 * kScales>());
        }
        if constexpr (t == kSlots - 1) {
          s_at += s_turn;
          s_turn = -s_turn;
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
  // Until the copies of all but the last two half stages have landed, in all waves, and what those were read for before
  // has left the stage's place.  (Behind a tile's end this waits for its stores too; counting them out gained nothing, as
  // all blocks end their tiles together and the stores are bound by the memory.)
  auto turn = [&]() __attribute__((always_inline)) {
    wait_vmem<kFirst + kCopies>();
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
  };

  GemmPlace p = place(walk.first);
  copy_from(source(p));
  unroll<kFirst>(copy_first);
  unroll<kCopies>(copy_second);
  copy_next();
  if (g.kb == 1) copy_zeros();
  wait_vmem<0>();
  __syncthreads();
  unroll<kFirst>(copy_first);
  unroll<kCopies>(copy_second);
  copy_next();
  unroll<F - 2>([&](auto qc) __attribute__((always_inline)) { read_part(std::integral_constant<int, 0>(), qc); });
  unroll<2>([&](auto ec) __attribute__((always_inline)) { read(std::integral_constant<int, F / 2 - 1>(), ec, spare); });
  unroll<F>([&](auto qc) __attribute__((always_inline)) { read_part(std::integral_constant<int, F>(), qc); });
  unroll<2 * kScales>(read_scale);
  unroll<2 * kScales>(take_scale);
  s_at += s_turn;
  s_turn = -s_turn;

  for (int item = walk.first; item < walk.last; item += walk.step) {
    const GemmPlace next = place(item + walk.step < walk.last ? item + walk.step : item);
    const Source next_source = source(next);
    if constexpr (!kShared) copy_bias(p.n0 + wn);
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int k = 0; k < F; ++k) acc[i][k] = f32x4_t{};
    hold_sums();
#pragma unroll 1
    for (int left = max(p.k1 - p.k0, 2); left > 0; --left) {  // a second stage of zeros where there is one block
      if (left <= 2) {  // here, not where they are used: a branch between the halves would let instructions sink past it
        if (left == 2) copy_from(next_source);
        else if (g.kb == 1) copy_zeros();
      }
#pragma unroll
      for (int i = 0; i < kScales; ++i) {
        sa[i] = sa1[i];
        sb[i] = sb1[i];
      }
      turn();
      half_stage(first);
      turn();
      half_stage(second);
      copy_next();
    }
    hold_sums();
    float bias[kScales];
    if constexpr (!kShared) read_bias(bias);
    const int m0 = p.m0 + wm, n0 = p.n0 + wn;
    if constexpr (kShared || C == kRowF32) {
      store_rows32<kShared>(g, acc, m0, n0, p.split, bias);
    } else {
      store_rows16<C, ACT>(g, acc, m0, n0, bias);
    }
    p = next;
  }
  wait_vmem<0>();  // no copy may land in LDS that is another block's by then
}

// Launches of the instances, each compiled in one of the fp8_gemm_*.hip files.
void launch_gemm_256(const GemmArgs& g, int a_type, int c, hipStream_t s);        // c: a 16-bit type or kShare
void launch_gemm_256_e5m2(const GemmArgs& g, int c, hipStream_t s);
void launch_gemm_128(const GemmArgs& g, int a_type, int c, hipStream_t s);        // any c

}  // namespace svoo
