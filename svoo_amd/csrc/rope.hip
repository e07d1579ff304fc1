// Rotary positions on several axes behind an RMS norm, with the backward pass.
//   n = x rstd w,  rstd = 1 / sqrt(mean(x^2) + eps) over a token's whole row or each head (or n = x without a norm)
//   pair (a, b) at angle t = p theta^(-2j / d) of its axis:  y = (a cos t - b sin t, a sin t + b cos t)
//   backward  g = the inverse turn of dy,  u = g w,  dx = rstd (u - x rstd^2 mean(u x)),  dw = sum g x rstd
// What bounds it: memory; forward reads x and writes y once, backward reads x and dy and writes dx once.  A row stays in the
// registers of its lanes as it lies in memory, and the two sums of the backward pass cross the lanes together.
//
// Lanes: ceil(D / 8) of them hold a head, four pairs each, and a wave as many whole heads as fit: a lane's columns lie at the
// same place of every head it sees, so its angles are those of one place.  Angles are whole turns in doubles (a position of
// 10^5 times a rate keeps 30 bits behind the point), reduced to an eighth of a turn and rounded to fp32 there.
//
// bf16, 128 channels, a norm over the row: 32760 x 12 heads 37 us (5.4 TB/s) forward and 61 (4.9) backward, 75600 x 40 heads
// 295 (5.2) and 450 (5.2); backward straight after forward, whose results are still being written out of the caches, 530.
#include <algorithm>
#include <type_traits>

#include "colsums.h"

namespace svoo {

constexpr int kMaxAxes = 4;
constexpr int kMaxHeadDim = 512;
enum PosType { kPosGrid = 0, kPosI32 = 1, kPosI64 = 2, kPosF32 = 3 };
enum NormOver { kNormNone = 0, kNormRow = 1, kNormHead = 2 };

struct RopeArgs {
  const void* x;  // [batch][rows][heads][d], element strides, contiguous columns
  long long x_batch, x_row, x_head;
  const void* dy;  // backward
  long long dy_batch, dy_row, dy_head;
  void* y;         // forward: y, backward: dx; [batch][rows][heads][d] contiguous
  const void* w;   // row norm: [heads * d], head norm: [d], or null
  int w_type;
  float* partial;  // backward: [blocks][heads * d or d] or null
  const void* pos; // [batch or 1][rows][axes]
  int pos_type;
  long long pos_batch;
  unsigned batch, rows;
  int heads, d, axes;
  int axis_end[kMaxAxes];        // pairs up to and with this axis
  double neg_rate[kMaxAxes];     // -2 log2(theta) / channels of the axis
  unsigned grid[kMaxAxes], grid_rows;
  int start[kMaxAxes];
  float eps;
  int lanes, heads_per_wave;     // of a head; of a wave
  unsigned head_blocks, head_step;  // head kernel: items a token is cut into, heads of one
};

// cos and sin of t whole turns.
__device__ __forceinline__ float2 turn_of(double t) {
  const double quarter = t * 4.0;
  const double q = __builtin_rint(quarter);
  const float x = (float)((quarter - q) * 1.5707963267948966);  // |x| <= pi / 4
  // the Taylor series; what is left out is below 2^-28 of the result
  const float z = x * x;
  const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), x);
  const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.0f);
  const int k = (int)(long long)(q - 4.0 * __builtin_floor(q * 0.25));  // 0 .. 3
  const float cs = k & 1 ? s : c, sn = k & 1 ? c : s;
  return make_float2(k == 1 || k == 2 ? -cs : cs, k >= 2 ? -sn : sn);
}

// Pair j's axis and its turns per position step.
struct PairRate {
  int axis;
  double turns;
};
__device__ __forceinline__ PairRate pair_rate(const RopeArgs& a, int j) {
  PairRate r = {0, 0.0};
  int from = 0;
#pragma unroll
  for (int i = 0; i < kMaxAxes; ++i) {
    if (i < a.axes) {
      if (j >= from && j < a.axis_end[i]) r = {i, exp2(a.neg_rate[i] * (double)(j - from)) * 0.15915494309189535};
      from = a.axis_end[i];
    }
  }
  return r;  // channels behind the last axis are not turned
}
__device__ __forceinline__ double position(const RopeArgs& a, unsigned batch, unsigned row, int axis) {
  if (a.pos_type == kPosGrid) {
    if (row >= a.grid_rows) return 0.0;  // tokens behind the grid
    unsigned n = row, p = 0;
    int start = 0;
#pragma unroll
    for (int i = kMaxAxes - 1; i >= 0; --i) {
      if (i < a.axes) {
        const unsigned g = a.grid[i], at = n % g;
        n /= g;
        if (i == axis) {
          p = at;
          start = a.start[i];
        }
      }
    }
    return (double)p + (double)start;
  }
  const long long i = (long long)batch * a.pos_batch + (long long)row * a.axes + axis;
  if (a.pos_type == kPosI32) return (double)((const int32_t*)a.pos)[i];
  if (a.pos_type == kPosI64) return (double)((const long long*)a.pos)[i];
  return (double)((const float*)a.pos)[i];
}

// Four pairs of a head as they lie in memory: eight neighbours, or four from each half of the head.
template <int T, bool kHalves>
struct Unit {
  u32x4_t v[T == kRowF32 ? 2 : 1];
  static constexpr int kSize = T == kRowF32 ? 4 : 2;

  // np: pairs of the unit that are within the head (4, fewer in its last unit, 0 or less: none).
  __device__ __forceinline__ void load(const void* p, long long head, int u, int half, int np) {
#pragma unroll
    for (int h = 0; h < (T == kRowF32 ? 2 : 1); ++h) v[h] = u32x4_t{0, 0, 0, 0};
    const char* at = (const char*)p + head * kSize;
    if (np >= 4) {
      if (!kHalves) {
        v[0] = ((const Dwords4*)(at + 8 * u * kSize))->v;
        if (T == kRowF32) v[T == kRowF32 ? 1 : 0] = ((const Dwords4*)(at + 8 * u * kSize + 16))->v;
      } else if (T == kRowF32) {
        v[0] = ((const Dwords4*)(at + 4 * u * kSize))->v;
        v[T == kRowF32 ? 1 : 0] = ((const Dwords4*)(at + (half + 4 * u) * kSize))->v;
      } else {
        const Dwords2 lo = *(const Dwords2*)(at + 4 * u * kSize), hi = *(const Dwords2*)(at + (half + 4 * u) * kSize);
        v[0] = u32x4_t{lo.v[0], lo.v[1], hi.v[0], hi.v[1]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = (kHalves ? e % 4 : e / 2) < np;
        const int col = kHalves ? (e / 4) * half + 4 * u + e % 4 : 8 * u + e;
        if (!in) continue;
        if (T == kRowF32) v[T == kRowF32 ? e / 4 : 0][e % 4] = ((const uint32_t*)at)[col];
        else v[0][e / 2] |= (uint32_t)((const uint16_t*)at)[col] << (16 * (e & 1));
      }
    }
  }
  __device__ __forceinline__ float at(int e) const {
    if (T == kRowF32) return __uint_as_float(v[T == kRowF32 ? e / 4 : 0][e % 4]);
    if (T == kRowBf16) return __uint_as_float(e & 1 ? v[0][e / 2] & 0xffff0000u : v[0][e / 2] << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[0][e / 2] >> (16 * (e & 1))));
  }
  // A pair's two values of f, by index.
  static __device__ __forceinline__ int first(int i) { return kHalves ? i : 2 * i; }
  static __device__ __forceinline__ int second(int i) { return kHalves ? 4 + i : 2 * i + 1; }
  static __device__ __forceinline__ void store(void* p, long long head, int u, int half, int np, const float (&f)[8]) {
    if (!kHalves) {
      store_row8<T, false>(p, head + 8 * u, 2 * np, f);
      return;
    }
    if (np <= 0) return;
    if (T == kRowF32 && np >= 4) {
      ((Dwords4*)((float*)p + head + 4 * u))->v = u32x4_t{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
      ((Dwords4*)((float*)p + head + half + 4 * u))->v = u32x4_t{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
    } else if (T != kRowF32 && np >= 4) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = T == kRowBf16 ? cvt_pk_bf16(f[2 * e], f[2 * e + 1])
                             : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * e]) |
                                   ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * e + 1]) << 16);
      *(Dwords2*)((uint16_t*)p + head + 4 * u) = Dwords2{{w[0], w[1]}};
      *(Dwords2*)((uint16_t*)p + head + half + 4 * u) = Dwords2{{w[2], w[3]}};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e % 4 < np) set_row_elem(p, T, head + (e / 4) * half + 4 * u + e % 4, f[e]);
    }
  }
};
template <bool kHalves>
__device__ __forceinline__ int unit_col(int u, int e, int half) {  // within the head
  return kHalves ? (e / 4) * half + 4 * u + e % 4 : 8 * u + e;
}

// ---------------------------------------------------------------- a norm over the whole row: one wave or four a token
// Angles: each lane turns one pair a row (two or more where heads have over 128 channels) and leaves cos and sin in LDS for
// all heads; the next row's while this one's sums cross the lanes.
// A wave takes a row alone where its registers hold it, else the block's four share one and meet in LDS: 32760 x 12 heads 37
// us forward and 61 backward alone, 73 and 133 shared; 75600 x 40 heads forward 297 and 306.  Backward, 40 heads alone leave
// two waves a SIMD: 590 us of 540 shared, with a forward pass in front.
template <int T, int WPR, int NC, bool kHalves, bool kGrad>
__global__ void __launch_bounds__(256) rope_row_kernel(RopeArgs a) {
  constexpr int kGroups = 4 / WPR, kTpr = WPR * kWave;  // rows of a block at a time
  __shared__ f32x4_t params[2][NC * kTpr];  // the weight: half of a unit, chunk, lane
  extern __shared__ float2 tables[];        // [kGroups][2][d / 2]
  __shared__ float2 scratch[2 * (WPR > 1 ? WPR : 1)];
  __shared__ float sums[kGrad && kGroups > 1 ? (kGroups - 1) * 8 * kWave : 1];
  using U = Unit<T, kHalves>;
  const int t = threadIdx.x % kTpr, group = threadIdx.x / kTpr, lane = threadIdx.x % kWave, wave = t / kWave;
  const int half = a.d / 2, u = lane % a.lanes, in_wave = lane / a.lanes;
  const int np = in_wave < a.heads_per_wave ? half - 4 * u : 0;
  const int cols = a.heads * a.d;
  auto head_of = [&](int c) { return (c * WPR + wave) * a.heads_per_wave + in_wave; };
  for (int i = threadIdx.x; i < NC * kTpr; i += blockDim.x) {
    const int c = i / kTpr, tt = i % kTpr, l = tt % kWave, iw = l / a.lanes;
    const int head = (c * WPR + tt / kWave) * a.heads_per_wave + iw, uu = l % a.lanes;
    const bool in = iw < a.heads_per_wave && head < a.heads;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool has = in && (kHalves ? e % 4 : e / 2) < half - 4 * uu;
      params[e / 4][i][e % 4] = has && a.w != nullptr ? row_elem(a.w, a.w_type, (long long)head * a.d + unit_col<kHalves>(uu, e, half)) : has ? 1.0f : 0.0f;
    }
  }
  const float inv = 1.0f / (float)cols;
  const unsigned step = gridDim.x * kGroups, total = a.batch * a.rows;
  float2* table = tables + group * 2 * half;
  // this thread's pairs of the tables: t, t + kTpr, ..
  PairRate rate[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) rate[k] = pair_rate(a, t + k * kTpr);
  auto fill = [&](unsigned r, int which) __attribute__((always_inline)) {
    const unsigned b = r / a.rows, row = r % a.rows;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = t + k * kTpr;
      if (j < half) table[which * half + j] = turn_of(rate[k].turns * position(a, b, row, rate[k].axis));
    }
    for (int j = t + 2 * kTpr; j < half; j += kTpr) {
      const PairRate pr = pair_rate(a, j);
      table[which * half + j] = turn_of(pr.turns * position(a, b, row, pr.axis));
    }
  };
  float dw[kGrad ? NC : 1][8];
#pragma unroll
  for (int c = 0; c < (kGrad ? NC : 1); ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = 0.0f;
  unsigned r = blockIdx.x * kGroups + group;
  // Every thread runs as many rounds as the block's first rows need: the barriers are the block's.
  const unsigned first = blockIdx.x * kGroups;
  const unsigned rounds = first < total ? (total - first + step - 1) / step : 0;
  if (r < total) fill(r, 0);
  __syncthreads();
  int which = 0, swap = 0;
  for (unsigned round = 0; round < rounds; ++round, r += step, which ^= 1) {
    const bool on = r < total;
    const unsigned b = on ? r / a.rows : 0, row = on ? r % a.rows : 0;
    U x[NC], dy[kGrad ? NC : 1];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int head = head_of(c), n = on && head < a.heads ? np : 0;
      x[c].load(a.x, (long long)b * a.x_batch + (long long)row * a.x_row + (long long)head * a.x_head, u, half, n);
      if (kGrad)
        dy[kGrad ? c : 0].load(a.dy, (long long)b * a.dy_batch + (long long)row * a.dy_row + (long long)head * a.dy_head, u, half, n);
    }
    float2 cs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = i < np ? table[which * half + 4 * u + i] : make_float2(1.0f, 0.0f);
    if (r + step < total) fill(r + step, which ^ 1);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s1 = fmaf(x[c].at(e), x[c].at(e), s1);
      if (kGrad) {
        const f32x4_t w0 = params[0][c * kTpr + t], w1 = params[1][c * kTpr + t];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = U::first(i), q = U::second(i);
          const float da = dy[kGrad ? c : 0].at(p), db = dy[kGrad ? c : 0].at(q);
          const float ga = fmaf(da, cs[i].x, db * cs[i].y), gb = fmaf(db, cs[i].x, -da * cs[i].y);
          s2 = fmaf(ga * (p < 4 ? w0[p & 3] : w1[p & 3]), x[c].at(p), s2);
          s2 = fmaf(gb * (q < 4 ? w0[q & 3] : w1[q & 3]), x[c].at(q), s2);
        }
      }
    }
    row_sums<kTpr>(s1, s2, scratch, swap);
    const float rstd = 1.0f / sqrtf(fmaf(s1, inv, a.eps));
    const float m = s2 * inv * rstd * rstd;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int head = head_of(c), n = on && head < a.heads ? np : 0;
      const long long to = ((long long)b * a.rows + row) * cols + (long long)head * a.d;
      const f32x4_t w0 = params[0][c * kTpr + t], w1 = params[1][c * kTpr + t];
      float out[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = U::first(i), q = U::second(i);
        const float wp = p < 4 ? w0[p & 3] : w1[p & 3], wq = q < 4 ? w0[q & 3] : w1[q & 3];
        if (!kGrad) {
          const float na = x[c].at(p) * rstd * wp, nb = x[c].at(q) * rstd * wq;
          out[p] = fmaf(na, cs[i].x, -nb * cs[i].y);
          out[q] = fmaf(na, cs[i].y, nb * cs[i].x);
        } else {
          const float da = dy[kGrad ? c : 0].at(p), db = dy[kGrad ? c : 0].at(q);
          const float ga = fmaf(da, cs[i].x, db * cs[i].y), gb = fmaf(db, cs[i].x, -da * cs[i].y);
          out[p] = rstd * fmaf(-m, x[c].at(p), ga * wp);
          out[q] = rstd * fmaf(-m, x[c].at(q), gb * wq);
          dw[kGrad ? c : 0][p] = fmaf(ga, n > i ? x[c].at(p) * rstd : 0.0f, dw[kGrad ? c : 0][p]);
          dw[kGrad ? c : 0][q] = fmaf(gb, n > i ? x[c].at(q) * rstd : 0.0f, dw[kGrad ? c : 0][q]);
        }
      }
      if (a.y != nullptr) U::store(a.y, to, u, half, n, out);
    }
    if (WPR == 1) __syncthreads();  // the next row's table; row_sums is one for rows of four waves
  }
  if (!kGrad || a.partial == nullptr) return;
#pragma unroll
  for (int c = 0; c < (kGrad ? NC : 1); ++c) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = dw[c][e];
    if (kGroups > 1) {
      __syncthreads();
      if (group > 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[((group - 1) * 8 + e) * kWave + lane] = v[e];
      __syncthreads();
      if (group == 0)
        for (int k = 0; k < kGroups - 1; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += sums[(k * 8 + e) * kWave + lane];
    }
    const int head = head_of(c);
    if (group == 0 && head < a.heads)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((kHalves ? e % 4 : e / 2) < np)
          a.partial[(size_t)blockIdx.x * cols + (long long)head * a.d + unit_col<kHalves>(u, e, half)] = v[e];
  }
}

// ---------------------------------------------------------------- a norm over each head, or none
// A head's lanes take a token and walk over its heads, kAhead of them in flight: the angles are made once.
template <int T, bool kHalves, bool kGrad, bool kNorm>
__global__ void __launch_bounds__(256) rope_head_kernel(RopeArgs a) {
  constexpr int kAhead = 4;
  __shared__ float sums[kGrad && kNorm ? 8 * 256 : 1];
  using U = Unit<T, kHalves>;
  const int lane = threadIdx.x % kWave, half = a.d / 2, u = lane % a.lanes, in_wave = lane / a.lanes;
  const int base = in_wave * a.lanes;
  const bool used = in_wave < a.heads_per_wave;
  const int np = used ? half - 4 * u : 0;
  const unsigned per_block = 4 * a.heads_per_wave, slot = threadIdx.x / kWave * a.heads_per_wave + in_wave;
  const unsigned long long items = (unsigned long long)a.batch * a.rows * a.head_blocks;
  const bool pow2 = (a.lanes & (a.lanes - 1)) == 0;
  auto head_sum = [&](float v) __attribute__((always_inline)) -> float {
    if (pow2) {
      for (int o = a.lanes / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
      return v;
    }
    float s = 0.0f;
    for (int o = 0; o < a.lanes; ++o) s += __shfl(v, base + o);
    return s;
  };
  PairRate rate[4];
  float w[8], dw[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) rate[i] = i < np ? pair_rate(a, 4 * u + i) : PairRate{0, 0.0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool has = (kHalves ? e % 4 : e / 2) < np;
    w[e] = !kNorm || !has || a.w == nullptr ? 1.0f : row_elem(a.w, a.w_type, unit_col<kHalves>(u, e, half));
    dw[e] = 0.0f;
  }
  const float inv = 1.0f / (float)a.d;
  // every lane of a wave runs the same rounds: sums cross the lanes
  for (unsigned long long first = (unsigned long long)blockIdx.x * per_block; first < items; first += (unsigned long long)gridDim.x * per_block) {
    const unsigned long long item = first + slot;
    const bool on = used && item < items;
    const unsigned tok = on ? (unsigned)(item / a.head_blocks) : 0, hb = on ? (unsigned)(item % a.head_blocks) : 0;
    const unsigned b = tok / a.rows, row = tok % a.rows;
    float2 cs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = on ? turn_of(rate[i].turns * position(a, b, row, rate[i].axis)) : make_float2(1.0f, 0.0f);
    for (unsigned h0 = 0; h0 < a.head_step; h0 += kAhead) {
      U x[kAhead], dy[kGrad ? kAhead : 1];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const unsigned head = hb * a.head_step + h0 + k;
        const int n = on && h0 + k < a.head_step && head < (unsigned)a.heads ? np : 0;
        if (!kGrad || kNorm) x[k].load(a.x, (long long)b * a.x_batch + (long long)row * a.x_row + (long long)head * a.x_head, u, half, n);
        if (kGrad) dy[kGrad ? k : 0].load(a.dy, (long long)b * a.dy_batch + (long long)row * a.dy_row + (long long)head * a.dy_head, u, half, n);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const unsigned head = hb * a.head_step + h0 + k;
        const int n = on && h0 + k < a.head_step && head < (unsigned)a.heads ? np : 0;
        float s1 = 0.0f, s2 = 0.0f, rstd = 1.0f, m = 0.0f, g[8];
        if (kGrad) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int p = U::first(i), q = U::second(i);
            const float da = dy[kGrad ? k : 0].at(p), db = dy[kGrad ? k : 0].at(q);
            g[p] = fmaf(da, cs[i].x, db * cs[i].y);
            g[q] = fmaf(db, cs[i].x, -da * cs[i].y);
          }
        }
        if (kNorm) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            s1 = fmaf(x[k].at(e), x[k].at(e), s1);
            if (kGrad) s2 = fmaf(g[e] * w[e], x[k].at(e), s2);
          }
          s1 = head_sum(s1);
          rstd = 1.0f / sqrtf(fmaf(s1, inv, a.eps));
          if (kGrad) m = head_sum(s2) * inv * rstd * rstd;
        }
        float out[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = U::first(i), q = U::second(i);
          if (!kGrad) {
            const float na = kNorm ? x[k].at(p) * rstd * w[p] : x[k].at(p), nb = kNorm ? x[k].at(q) * rstd * w[q] : x[k].at(q);
            out[p] = fmaf(na, cs[i].x, -nb * cs[i].y);
            out[q] = fmaf(na, cs[i].y, nb * cs[i].x);
          } else if (kNorm) {
            out[p] = rstd * fmaf(-m, x[k].at(p), g[p] * w[p]);
            out[q] = rstd * fmaf(-m, x[k].at(q), g[q] * w[q]);
            dw[p] = fmaf(g[p], i < n ? x[k].at(p) * rstd : 0.0f, dw[p]);
            dw[q] = fmaf(g[q], i < n ? x[k].at(q) * rstd : 0.0f, dw[q]);
          } else {
            out[p] = g[p];
            out[q] = g[q];
          }
        }
        if (a.y != nullptr)
          U::store(a.y, (((long long)b * a.rows + row) * a.heads + head) * a.d, u, half, n, out);
      }
    }
  }
  if (!kGrad || !kNorm || a.partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[kGrad && kNorm ? e * 256 + threadIdx.x : 0] = dw[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * a.lanes; i += 256) {  // one column a thread: the block's heads in their order
    const int uu = i / 8, e = i % 8;
    if ((kHalves ? e % 4 : e / 2) >= half - 4 * uu) continue;
    float s = 0.0f;
    for (int wv = 0; wv < 4; ++wv)
      for (int k = 0; k < a.heads_per_wave; ++k) s += sums[kGrad && kNorm ? e * 256 + wv * kWave + k * a.lanes + uu : 0];
    a.partial[(size_t)blockIdx.x * a.d + unit_col<kHalves>(uu, e, half)] = s;
  }
}

// Blocks: as many as are resident, for the gradients' partial rows two a CU.
static unsigned rope_blocks(long long tokens, int heads, int d, int norm, bool grad, unsigned* head_blocks, unsigned* head_step) {
  const int lanes = (d + 7) / 8, hpw = kWave / lanes;
  if (norm == kNormRow) {
    const long long groups = heads <= 3 * hpw || (!grad && heads <= 10 * hpw) ? 4 : 1;
    return (unsigned)std::min<long long>((tokens + groups - 1) / groups, grad ? 512 : 1024);
  }
  *head_step = (unsigned)std::min(heads, 16);
  *head_blocks = (unsigned)((heads + *head_step - 1) / *head_step);
  const long long items = tokens * *head_blocks;
  return (unsigned)std::min<long long>((items + 4 * hpw - 1) / (4 * hpw), grad && norm == kNormHead ? 1024 : 2048);
}

template <int T, bool kHalves, bool kGrad>
static void launch_row(const RopeArgs& a, unsigned blocks, hipStream_t s) {
  const int chunks1 = (a.heads + a.heads_per_wave - 1) / a.heads_per_wave;
  auto go = [&](auto wpr, auto nc) {
    constexpr int kWpr = decltype(wpr)::value, kNc = decltype(nc)::value;
    const size_t lds = (size_t)(4 / kWpr) * 2 * (a.d / 2) * sizeof(float2);
    hipLaunchKernelGGL((rope_row_kernel<T, kWpr, kNc, kHalves, kGrad>), dim3(blocks), dim3(256), lds, s, a);
  };
  using std::integral_constant;
  if (chunks1 <= 1) go(integral_constant<int, 1>(), integral_constant<int, 1>());
  else if (chunks1 <= 3) go(integral_constant<int, 1>(), integral_constant<int, 3>());
  else if (!kGrad && chunks1 <= 10) go(integral_constant<int, 1>(), integral_constant<int, kGrad ? 3 : 10>());
  else if (chunks1 <= 12) go(integral_constant<int, 4>(), integral_constant<int, 3>());
  else go(integral_constant<int, 4>(), integral_constant<int, 8>());
}

template <int T, bool kHalves, bool kGrad>
static void launch_rope(const RopeArgs& a, int norm, unsigned blocks, hipStream_t s) {
  if (norm == kNormRow) launch_row<T, kHalves, kGrad>(a, blocks, s);
  else if (norm == kNormHead) hipLaunchKernelGGL((rope_head_kernel<T, kHalves, kGrad, true>), dim3(blocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rope_head_kernel<T, kHalves, kGrad, false>), dim3(blocks), dim3(256), 0, s, a);
}
template <bool kGrad>
static void launch_rope(const RopeArgs& a, int type, int norm, bool halves, unsigned blocks, hipStream_t s) {
  if (type == kRowBf16) halves ? launch_rope<kRowBf16, true, kGrad>(a, norm, blocks, s) : launch_rope<kRowBf16, false, kGrad>(a, norm, blocks, s);
  else if (type == kRowF16) halves ? launch_rope<kRowF16, true, kGrad>(a, norm, blocks, s) : launch_rope<kRowF16, false, kGrad>(a, norm, blocks, s);
  else halves ? launch_rope<kRowF32, true, kGrad>(a, norm, blocks, s) : launch_rope<kRowF32, false, kGrad>(a, norm, blocks, s);
}

static int check_rope(const char* name, int type, long long batch, long long rows, int heads, int d, int norm, int axes,
                      const int* axis_channels, const double* theta, const int* grid, int pos_type, const void* pos,
                      int w_type, RopeArgs* a) {
  SVOO_REQUIRE(type >= 0 && type <= 2 && w_type >= 0 && w_type <= 2, SVOO_ERR_INVALID_ARG,
               "%s: element types %d %d (0 bf16, 1 fp16, 2 fp32)", name, type, w_type);
  SVOO_REQUIRE(batch >= 0 && rows >= 0 && heads > 0 && d > 0 && d % 2 == 0, SVOO_ERR_INVALID_ARG,
               "%s: batch=%lld rows=%lld heads=%d d=%d", name, batch, rows, heads, d);
  SVOO_REQUIRE(d <= kMaxHeadDim, SVOO_ERR_UNSUPPORTED, "%s: d=%d (2..%d)", name, d, kMaxHeadDim);
  SVOO_REQUIRE(norm >= 0 && norm <= 2, SVOO_ERR_INVALID_ARG, "%s: norm %d (0 none, 1 row, 2 head)", name, norm);
  a->lanes = (d + 7) / 8;
  a->heads_per_wave = kWave / a->lanes;
  SVOO_REQUIRE(norm != kNormRow || heads <= 32 * a->heads_per_wave, SVOO_ERR_UNSUPPORTED,
               "%s: a norm over rows of %d heads of %d (at most %d)", name, heads, d, 32 * a->heads_per_wave);
  SVOO_REQUIRE(heads <= 65536 && batch < (1ll << 31) && rows < (1ll << 31) && batch * rows < (1ll << 31), SVOO_ERR_UNSUPPORTED,
               "%s: %d heads of %lld x %lld tokens", name, heads, batch, rows);
  SVOO_REQUIRE(axes >= 1 && axes <= kMaxAxes, SVOO_ERR_INVALID_ARG, "%s: %d axes (1..%d)", name, axes, kMaxAxes);
  SVOO_REQUIRE(axis_channels && theta, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  SVOO_REQUIRE(pos_type >= 0 && pos_type <= 3, SVOO_ERR_INVALID_ARG,
               "%s: position type %d (0 grid, 1 int32, 2 int64, 3 fp32)", name, pos_type);
  int pairs = 0;
  unsigned long long cells = 1;
  for (int i = 0; i < axes; ++i) {
    SVOO_REQUIRE(axis_channels[i] >= 0 && axis_channels[i] % 2 == 0 && theta[i] > 0 && theta[i] < 1e300, SVOO_ERR_INVALID_ARG,
                 "%s: axis %d of %d channels, theta %g", name, i, axis_channels[i], theta[i]);
    pairs += axis_channels[i] / 2;
    SVOO_REQUIRE(pairs <= d / 2, SVOO_ERR_INVALID_ARG, "%s: axes of more than %d channels", name, d);
    a->axis_end[i] = pairs;
    a->neg_rate[i] = axis_channels[i] ? -2.0 * log2(theta[i]) / axis_channels[i] : 0.0;
    if (pos_type == kPosGrid) {
      SVOO_REQUIRE(grid && grid[i] > 0, SVOO_ERR_INVALID_ARG, "%s: grid of %d along axis %d", name, grid ? grid[i] : 0, i);
      a->grid[i] = (unsigned)grid[i];
      cells = std::min(cells * (unsigned)grid[i], 1ull << 32);
    }
  }
  a->grid_rows = (unsigned)std::min(cells, (1ull << 31) - 1);
  SVOO_REQUIRE(pos_type == kPosGrid || pos || batch * rows == 0, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  a->axes = axes;
  a->batch = (unsigned)batch;
  a->rows = (unsigned)rows;
  a->heads = heads;
  a->d = d;
  a->pos = pos;
  a->pos_type = pos_type;
  a->w_type = w_type;
  return SVOO_OK;
}

}  // namespace svoo

using namespace svoo;

extern "C" int svoo_axis_rope_fwd(const void* x, int type, long long x_batch_stride, long long x_row_stride,
                                  long long x_head_stride, long long batch, long long rows, int heads, int d, int norm,
                                  const void* w, int w_type, float eps, int axes, const int* axis_channels,
                                  const double* theta, const int* grid, const int* grid_start, const void* positions,
                                  int pos_type, long long pos_batch_stride, int halves, void* y, void* stream) {
  static const char* name = "svoo_axis_rope_fwd";
  RopeArgs a = {};
  if (const int rc = check_rope(name, type, batch, rows, heads, d, norm, axes, axis_channels, theta, grid, pos_type,
                                positions, w_type, &a))
    return rc;
  if (batch * rows == 0) return SVOO_OK;
  SVOO_REQUIRE(x && y, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  a.x = x;
  a.x_batch = x_batch_stride;
  a.x_row = x_row_stride;
  a.x_head = x_head_stride;
  a.y = y;
  a.w = w;
  a.eps = eps;
  a.pos_batch = pos_batch_stride;
  for (int i = 0; i < axes; ++i) a.start[i] = grid_start ? grid_start[i] : 0;
  const unsigned blocks = rope_blocks(batch * rows, heads, d, norm, false, &a.head_blocks, &a.head_step);
  launch_rope<false>(a, type, norm, halves != 0, blocks, (hipStream_t)stream);
  return check_launch(name);
}

extern "C" size_t svoo_axis_rope_bwd_workspace_size(long long batch, long long rows, int heads, int d, int norm) {
  if (batch <= 0 || rows <= 0 || heads <= 0 || d <= 0 || d > kMaxHeadDim || norm == kNormNone) return 0;
  unsigned hb, hs;
  return (size_t)rope_blocks(batch * rows, heads, d, norm, true, &hb, &hs) * (norm == kNormRow ? heads * d : d) * sizeof(float);
}

extern "C" int svoo_axis_rope_bwd(const void* dy, long long dy_batch_stride, long long dy_row_stride,
                                  long long dy_head_stride, const void* x, int type, long long x_batch_stride,
                                  long long x_row_stride, long long x_head_stride, long long batch, long long rows,
                                  int heads, int d, int norm, const void* w, int w_type, float eps, int axes,
                                  const int* axis_channels, const double* theta, const int* grid, const int* grid_start,
                                  const void* positions, int pos_type, long long pos_batch_stride, int halves, void* dx,
                                  void* dw, int dw_type, void* workspace, size_t ws_bytes, void* stream) {
  static const char* name = "svoo_axis_rope_bwd";
  RopeArgs a = {};
  if (const int rc = check_rope(name, type, batch, rows, heads, d, norm, axes, axis_channels, theta, grid, pos_type,
                                positions, w_type, &a))
    return rc;
  SVOO_REQUIRE(dw_type >= 0 && dw_type <= 2, SVOO_ERR_INVALID_ARG, "%s: element type %d (0 bf16, 1 fp16, 2 fp32)", name, dw_type);
  SVOO_REQUIRE(dw == nullptr || norm != kNormNone, SVOO_ERR_INVALID_ARG, "%s: a weight's gradient without a norm", name);
  if (batch * rows == 0) {
    SVOO_REQUIRE(!dw, SVOO_ERR_INVALID_ARG, "%s: a weight's gradient of no rows", name);
    return SVOO_OK;
  }
  if (!dx && !dw) return SVOO_OK;
  SVOO_REQUIRE(dy && (x || norm == kNormNone), SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  const size_t need = svoo_axis_rope_bwd_workspace_size(batch, rows, heads, d, norm);
  SVOO_REQUIRE(!dw || (workspace && ws_bytes >= need), SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)", name,
               ws_bytes, need);
  a.x = x;
  a.x_batch = x_batch_stride;
  a.x_row = x_row_stride;
  a.x_head = x_head_stride;
  a.dy = dy;
  a.dy_batch = dy_batch_stride;
  a.dy_row = dy_row_stride;
  a.dy_head = dy_head_stride;
  a.y = dx;
  a.w = w;
  a.eps = eps;
  a.pos_batch = pos_batch_stride;
  a.partial = dw ? (float*)workspace : nullptr;
  for (int i = 0; i < axes; ++i) a.start[i] = grid_start ? grid_start[i] : 0;
  const unsigned blocks = rope_blocks(batch * rows, heads, d, norm, true, &a.head_blocks, &a.head_step);
  launch_rope<true>(a, type, norm, halves != 0, blocks, (hipStream_t)stream);
  if (const int rc = check_launch(name)) return rc;
  if (!dw) return SVOO_OK;
  const int cols = norm == kNormRow ? heads * d : d;
  const ColSumsArgs c = {(const float*)workspace, 1, blocks, 1, cols, {dw, nullptr, nullptr}, {dw_type, 2, 2}, {0, 0, 0}};
  hipLaunchKernelGGL(column_sums_kernel, dim3((cols + kWave - 1) / kWave, 1, 1), dim3(1024), 0, (hipStream_t)stream, c);
  return check_launch(name);
}
