// Dense attention over heads that may share keys and values, with its backward pass: what the kernels share.
//   S = scale q k^T over the keys of a sequence,  L = logsumexp(S),  P = exp(S - L),  o = P v
//   backward  D = rowsum(do o),  dP = do v^T,  dS = P (dP - D),  dv = P^T do,  dq = scale dS k,  dk = scale dS^T q
// Queries from a sequence's length on have o = 0 and no gradient, keys from theirs on take no part; a query without keys has
// o = 0 and L = -inf.  A score of -inf has P = 0; a query that has keys but no other scores has no P: o and L are NaN.
//
// Every product is a 32 x 32 x 16 matrix instruction whose accumulator is the next product's operand as it lies: scores come
// out with one query (or key) per lane and 16 of the other side in its registers, which is the operand of the product that
// contracts that side, up to the order of the contracted positions; the other operand is read from LDS in the same order by
// gfx950's transposing read.  Rows behind a sequence's end are read as its last row, columns behind the head dim as zeros; rows
// of v and do there, which are multiplied by P = 0, become zeros too (an infinite last row would make 0 times inf).
#pragma once

#include <algorithm>
#include <type_traits>

#include "svoo_common.h"

namespace svoo {

enum DenseType { kDenseBf16 = 0, kDenseF16 = 1 };

// By type, padded head dim (64 or 128) and whether the head dim is that.
template <class F>
static void for_dense(int type, int d, F f) {
  using std::integral_constant;
  auto dims = [&](auto t) {
    if (d == 128) f(t, integral_constant<int, 128>(), std::true_type());
    else if (d > 64) f(t, integral_constant<int, 128>(), std::false_type());
    else if (d == 64) f(t, integral_constant<int, 64>(), std::true_type());
    else f(t, integral_constant<int, 64>(), std::false_type());
  };
  if (type == kDenseBf16) dims(integral_constant<int, kDenseBf16>());
  else dims(integral_constant<int, kDenseF16>());
}

struct DenseRows {  // [batch][heads][rows][d] by strides in elements, columns contiguous, rows at 16-byte addresses
  const uint16_t* p;
  long long batch, head, row;
};

struct DenseArgs {
  DenseRows q, k, v, o, dy;
  uint16_t* out;        // forward: o; backward: dq
  uint16_t* rest;       // forward: what o's rounding left, laid out as o, or null; backward: the same
  uint16_t *dk, *dv;    // contiguous [batch][rows][heads][d]
  float* lse;           // [batch][heads][sq]
  float* delta;         // the same: rowsum(do o)
  float* norms;         // fp16: the largest |do|^2 and |v|^2 of every kNormRows rows
  const int32_t *q_lens, *k_lens;  // [batch] or null
  float* part;          // partial results of shares, or null
  float4* part_ml;      // forward: maximum, sum, sum of the rounded P
  int batch, heads, kv_heads, group;  // group = heads / kv_heads
  int sq, sk, d;
  int splits;           // shares of the contracted length
  int tiles;            // of the rows that a block owns
  float scale, scale_log2;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A running maximum starts at the lowest number: from -inf, a tile whose scores are all -inf would have P = exp(-inf + inf), and
// the row would be NaN for good, whatever follows.
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kNormRows = 256;  // rows that share a maximum
// fp16's P runs to 2^14 in the backward pass, so that 1 / N of a long even row is a normal number
constexpr float kF16PShift = 14.0f;
// and in the forward pass from 2^12 of a running maximum to the type's end: with all its bits to 2^-26 of the largest, in steps of
// 2^-36 below.  With P = 1 at the maximum, keys 14 bits below it lost bits and those 25 below it were lost, which is all of o
// where the largest one's value is 0 (even keys at e^-16 and e^-17 of it: o 8% and 44% too large; at e^-18: o = 0).
constexpr float kF16Top = 12.0f;
// for maxima below 2^22: a step of those is a quarter at most.  From 2^26 on, with steps of 8, a maximum less 12 may come out 16
// lower, and P past the type's range.
constexpr float kF16TopWithin = 4194304.0f;

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

template <int T>
__device__ __forceinline__ f32x16_t mma(u32x4_t a, u32x4_t b, f32x16_t c) {
  if (T == kDenseBf16) return mfma32x32x16(as_bf16x8(a), as_bf16x8(b), c);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <int T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (T == kDenseBf16) return cvt_pk_bf16(lo, hi);
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}
// L of a row with keys, from its maximum and sum; NaN without a finite score.
__device__ __forceinline__ float row_lse(float m, float l) {
  return l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : __builtin_nanf("");
}
// c plus a pair's two values (P rounded: o is divided by the sum of what multiplied v, so that its weights sum to 1)
template <int T>
__device__ __forceinline__ float sum2(uint32_t w, float c) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if (T == kDenseBf16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), c, false);
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), c, false);
}
template <int T>
__device__ __forceinline__ float elem16(uint32_t w, int hi) {
  if (T == kDenseBf16) return __uint_as_float(hi ? w & 0xffff0000u : w << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w));
}

// Physical 16-byte chunk of logical chunk c in row r of a tile of DP columns (an involution for a given r).
template <int DP>
__device__ __forceinline__ int tile_swz(int r, int c) {
  return DP == 128 ? swz(r, c) : c ^ ((r >> 1) & 7);
}

__device__ __forceinline__ int seq_len(const int32_t* lens, int b, int most) {
  return lens == nullptr ? most : min(max(lens[b], 0), most);
}

// Rows row0 .. of a matrix into an LDS tile of kRows x DP by LDS DMA, issued by kWaves waves (this one the w-th); rows behind
// `last` repeat it.  A scalar base and 32-bit offsets: rows are below 2^24 bytes apart.  Columns from d on are left as
// they are (tile_clear).
template <int DP, bool kFull, int kRows, int kWaves>
__device__ __forceinline__ void tile_dma(const uint16_t* base, long long row_stride, int row0, int last, int d, uint16_t* tile,
                                         int w, int lane) {
  constexpr int kChunks = DP / 8, kIt = kRows * kChunks / (64 * kWaves), kEach = 64 / kChunks;  // rows of a copy
  w = __builtin_amdgcn_readfirstlane(w);
  const int first = min(row0, last), most = last - first;
  const char* from = (const char*)(base + first * row_stride);
  const uint32_t step = (uint32_t)row_stride * 2;
  uint32_t l = lane;
  __asm__ volatile("" : "+v"(l));  // places made here: kept from tile to tile they take registers that the sums need
  // row n kEach + l / kChunks has chunk l % kChunks where the swizzle of the lane's part of the row and of n's put it
  const uint32_t row = l / kChunks, chunk = l % kChunks ^ (DP == 128 ? row << 2 : l / 16);
#pragma unroll
  for (int j = 0; j < kIt; ++j) {
    const uint32_t n = w * kIt + j, c = chunk ^ (DP == 128 ? n & 3 : (n & 1) << 2);
    if (kFull || c * 8 < (uint32_t)d) lds_dma16(from + (__umul24(min(n * kEach + row, (uint32_t)most), step) + c * 16), tile + n * 64 * 8);
  }
}
// Rows n .. of a tile as zeros, each wave those that it copied, once its copies are there.
template <int DP, int kRows, int kWaves>
__device__ __forceinline__ void tile_end(uint16_t* tile, int n, int w, int lane) {
  constexpr int kEach = kRows / kWaves * DP / 8;  // 16-byte chunks of a wave
  w = __builtin_amdgcn_readfirstlane(w);
#pragma unroll
  for (int i = 0; i < kEach; i += 64)
    if (w * kEach + i + lane >= n * (DP / 8)) ((u32x4_t*)tile)[w * kEach + i + lane] = u32x4_t{0, 0, 0, 0};
}
// Tiles with columns that no copy fills, once: zeros.
template <int DP, int kThreads, int kElems>
__device__ __forceinline__ void tile_clear(uint16_t* tiles, int d) {
  if (d == DP) return;
  for (int i = threadIdx.x; i < kElems / 8; i += kThreads) ((u32x4_t*)tiles)[i] = u32x4_t{0, 0, 0, 0};
}

// A lane's operand of a row's columns: positions 16 s + 8 h .. + 7 for s = 0 .. DP / 16 - 1.
template <int DP, bool kFull>
__device__ __forceinline__ void load_operand(const uint16_t* row, int d, int h, u32x4_t (&op)[DP / 16]) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int c = 16 * s + 8 * h;
    op[s] = kFull || c < d ? *(const u32x4_t*)(row + c) : u32x4_t{0, 0, 0, 0};
  }
}

// Where a lane reads a tile: row operands of rows 0 .. 31 (the swizzle repeats every 16 rows), and the transposing reads of
// rows 0 .. 15 (first and second four a lane half contracts) for the 32 columns db.  The swizzle is an exclusive or of chunk
// numbers, so the other places are the first one's with a constant.
template <int DP>
struct TileReads {
  int row0, lo0, hi0;
  __device__ __forceinline__ void init(int lane) {
    const int h = lane / 32, l32 = lane % 32, grp = lane / 16, gl = lane % 16;
    row0 = l32 * DP + tile_swz<DP>(l32, h) * 8;
    const int r0 = 4 * (grp / 2) + gl / 4, c = 2 * (grp % 2) + (gl % 4) / 2, e0 = 4 * (gl % 2);
    lo0 = r0 * DP + tile_swz<DP>(r0, c) * 8 + e0;
    hi0 = (r0 + 8) * DP + tile_swz<DP>(r0 + 8, c) * 8 + e0;
  }
  // Places are made from here on: kept from step to step they take registers that the sums need.
  __device__ __forceinline__ void forget() { __asm__ volatile("" : "+v"(row0), "+v"(lo0), "+v"(hi0)); }
  __device__ __forceinline__ u32x4_t row(const uint16_t* tile, int s) const { return *(const u32x4_t*)(tile + (row0 ^ (16 * s))); }
  __device__ __forceinline__ u32x4_t cols(const uint16_t* tile, int db) const {
    const uint2 a = ds_read_tr16_b64(tile + (lo0 ^ (32 * db))), b = ds_read_tr16_b64(tile + (hi0 ^ (32 * db)));
    return u32x4_t{a.x, a.y, b.x, b.y};
  }
};

// The blocks of a launch, so that consecutive ones of a head (which read the same rows) run on one XCD: workgroups go round
// robin over the 8 XCDs.
__device__ __forceinline__ unsigned xcd_block(unsigned bid, unsigned total) {
  const unsigned each = (total + 7) / 8;
  return (bid % 8) * each + bid / 8;
}

// Where four rounds of blocks or more walk over few tiles, the first round's blocks (one a CU) start apart, over about the time
// of a block (15 us at most): else all of them read their rows at the same time, then all compute, and so to the end.  bf16,
// 128 columns, forward and dq without and with it: 12 x 22000 x 512 105 and 95, 120 and 108 us; 12 x 32760 x 512 133 and 128,
// 181 and 168, x 64 67 and 63, 79 and 77, x 1024 212 and 211, 301 and 294; 64 columns, 16 x 32760 x 512 115 and 116, 143 and
// 142, 24 x 75600 x 256 280 and 274.  It is kept where it wins nothing, at 64 columns and at 16 tiles, since it costs nothing there.
// Above 16 tiles a walk nothing is won (12 x 32760 x 4096 711 and 717 us), and delays twice as long lost 5% at 1024.
template <int DP>
__device__ __forceinline__ void start_apart(unsigned total, int ntiles) {
  if (blockIdx.x >= 256 || total < 1024 || ntiles > 16) return;
  const int n = (int)blockIdx.x / 8 * min(ntiles, 8) * DP / 128;
  for (int i = 0; i < n; ++i) __builtin_amdgcn_s_sleep(2);
}

// Four values to 16 bits, and what that leaves of them.
template <int T>
__device__ __forceinline__ uint2 pack4(f32x4_t v) { return make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])); }
template <int T>
__device__ __forceinline__ f32x4_t rest4(f32x4_t v, uint2 w) {
  return f32x4_t{v[0] - elem16<T>(w.x, 0), v[1] - elem16<T>(w.x, 1), v[2] - elem16<T>(w.y, 0), v[3] - elem16<T>(w.y, 1)};
}
// Two groups of eight columns, of which each lane of a pair (l, l + 32) holds four: the first group whole in the lower lane,
// the second in the upper one.
__device__ __forceinline__ u32x4_t join_halves(uint2 a, uint2 b) {
  const auto x = __builtin_amdgcn_permlane32_swap(a.x, b.x, false, false), y = __builtin_amdgcn_permlane32_swap(a.y, b.y, false, false);
  return u32x4_t{x[0], y[0], x[1], y[1]};
}
// acc [columns][row of this lane] to a contiguous row of 16-bit elements, both lanes of a row together.
template <int T, int DP, bool kFull>
__device__ __forceinline__ void store_row16(uint16_t* row, uint16_t* rest, const f32x16_t (&acc)[DP / 32], int d, int h,
                                            float by) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {
      const int c = 32 * db + 16 * pair + 8 * h;
      f32x4_t v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = acc[db][8 * pair + 4 * i + e] * by;
      const uint2 a = pack4<T>(v[0]), b = pack4<T>(v[1]);
      const u32x4_t w = join_halves(a, b);
      if (kFull || c < d) *(u32x4_t*)(row + c) = w;
      if (rest != nullptr) {
        const u32x4_t r = join_halves(pack4<T>(rest4<T>(v[0], a)), pack4<T>(rest4<T>(v[1], b)));
        if (kFull || c < d) *(u32x4_t*)(rest + c) = r;
      }
    }
}
template <int DP, bool kFull>
__device__ __forceinline__ void store_row32(float* row, const f32x16_t (&acc)[DP / 32], int d, int h) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int c = 32 * db + 8 * r4 + 4 * h;
      if (kFull || c < d) *(f32x4_t*)(row + c) = f32x4_t{acc[db][4 * r4], acc[db][4 * r4 + 1], acc[db][4 * r4 + 2], acc[db][4 * r4 + 3]};
    }
}

// dense.hip
int dense_shares(long long blocks, long long units, long long bytes);
bool dense_rows_ok(const DenseRows& m);
int check_dense(const char* name, int type, int batch, int heads, int kv_heads, int sq, int sk, int d);

}  // namespace svoo
