// Dense attention: the backward pass, as two kernels that compute the probabilities again, so that every sum has a fixed order:
// one owns queries and walks over the keys (dq), one owns keys and walks over the queries of the heads that share them
// (dk, dv).  That is seven products where one kernel with atomic sums would take five.
#include "dense.h"

namespace svoo {

constexpr int kBwdWaves = 8, kBwdRows = kBwdWaves * 32, kBwdTile = 64;

// delta = rowsum(do o), with o to twice its bits where its rounding is known: an error of D enters every dS of a row with one
// sign and is multiplied by the mean key (dq 0.0035 off at 1000 keys with it, 0.0026 without, 0.0017 of that the result's own
// rounding).  For fp16 the largest |do|^2 (and |v|^2) of every kNormRows rows.
// Memory bounds it: 12 x 32760 rows of 128 columns in 61 us, 4.9 TB/s; 24888 rows of 64 in 9 us, 14 with half the threads.
constexpr int kDeltaThreads = 512;
template <int T>
__global__ void __launch_bounds__(kDeltaThreads) dense_delta_kernel(DenseArgs a, int q_blocks, int v_blocks) {
  constexpr int kWaves = kDeltaThreads / kWave, kAtOnce = kDeltaThreads / 16;
  __shared__ float top[kWaves];
  const bool is_v = (int)blockIdx.x >= q_blocks;
  const int n = is_v ? blockIdx.x - q_blocks : blockIdx.x, per = ((is_v ? a.sk : a.sq) + kNormRows - 1) / kNormRows;
  const int heads = is_v ? a.kv_heads : a.heads, bh = n / per, b = bh / heads, head = bh % heads;
  const int rows = is_v ? a.sk : a.sq, len = is_v ? seq_len(a.k_lens, b, a.sk) : seq_len(a.q_lens, b, a.sq);
  const DenseRows m = is_v ? a.v : a.dy;
  const int c = threadIdx.x % 16 * 8, r0 = n % per * kNormRows + threadIdx.x / 16;
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < kNormRows / kAtOnce; ++i) {
    const int row = r0 + kAtOnce * i;
    float dot = 0.0f, sq = 0.0f;
    if (row < len && c < a.d) {
      const u32x4_t x = *(const u32x4_t*)(m.p + (long long)b * m.batch + (long long)head * m.head + (long long)row * m.row + c);
      u32x4_t y = {0, 0, 0, 0}, z = y;
      if (!is_v) {
        y = *(const u32x4_t*)(a.o.p + (long long)b * a.o.batch + (long long)head * a.o.head + (long long)row * a.o.row + c);
        if (a.rest != nullptr) z = *(const u32x4_t*)(a.rest + (((size_t)b * a.sq + row) * a.heads + head) * a.d + c);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = elem16<T>(x[e / 2], e & 1);
        dot = fmaf(u, elem16<T>(y[e / 2], e & 1) + elem16<T>(z[e / 2], e & 1), dot);
        if (T == kDenseF16) sq = fmaf(u, u, sq);
      }
    }
    for (int o = 8; o > 0; o >>= 1) {
      dot += __shfl_xor(dot, o);
      if (T == kDenseF16) sq += __shfl_xor(sq, o);
    }
    if (!is_v && c == 0 && row < rows) a.delta[(size_t)bh * a.sq + row] = dot;
    most = fmaxf(most, sq);
  }
  if (T != kDenseF16) return;
  for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
  if (threadIdx.x % kWave == 0) top[threadIdx.x / kWave] = most;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < kWaves; ++i) most = fmaxf(most, top[i]);
  a.norms[blockIdx.x] = most;
}

// fp16's dS is kept as dS 2^e: |dP - D| is at most 2 |do| |v|, and e takes the largest of that to 2^14 .. 2^15, so that dS is a
// normal number down to 2^-29 of its bound.  The same for the heads that share keys.
__device__ __forceinline__ float f16_exponent(const DenseArgs& a, int b, int kv, float* scratch) {
  const int nq = (a.sq + kNormRows - 1) / kNormRows, nk = (a.sk + kNormRows - 1) / kNormRows;
  const float* dy = a.norms + ((size_t)b * a.heads + (size_t)kv * a.group) * nq;
  const float* v = a.norms + (size_t)a.batch * a.heads * nq + ((size_t)b * a.kv_heads + kv) * nk;
  float md = 0.0f, mv = 0.0f;
  for (int i = threadIdx.x; i < a.group * nq; i += blockDim.x) md = fmaxf(md, dy[i]);
  for (int i = threadIdx.x; i < nk; i += blockDim.x) mv = fmaxf(mv, v[i]);
  for (int o = 32; o > 0; o >>= 1) {
    md = fmaxf(md, __shfl_xor(md, o));
    mv = fmaxf(mv, __shfl_xor(mv, o));
  }
  const int w = threadIdx.x / kWave, waves = blockDim.x / kWave;
  if (threadIdx.x % kWave == 0) {
    scratch[w] = md;
    scratch[waves + w] = mv;
  }
  __syncthreads();
  for (int i = 0; i < waves; ++i) {
    md = fmaxf(md, scratch[i]);
    mv = fmaxf(mv, scratch[waves + i]);
  }
  const float most = 2.0f * sqrtf(md) * sqrtf(mv);
  if (!(most > 0.0f && most < INFINITY)) return 0.0f;
  return fminf(fmaxf(14.0f - (float)((int)(__float_as_uint(most) >> 23) - 127), -60.0f), 60.0f);
}

// Both kernels run 8 waves, two on each SIMD.  The waves of a SIMD belong to two groups that alternate, half a step apart,
// between a step's matrix work (the sums of step u, then the scores of step u + 1) and the arithmetic on the scores of the
// next, so that matrix and vector units are busy at the same time: without the two groups, waves of a block that meet at
// every tile's barrier do the same thing at the same time, and a step takes the sum of both (dq 10.4 ms at 12 x 32760 x 128
// where the two waves of a SIMD belong to one group, 8.5 so).
// A step is 32 rows of the other side, half a tile; group B copies tile t + 1 during step 2 t, into the buffer of tile t - 1.
// Matrix work goes first where both want to issue (7.4 ms and 7.2 of dq at full clocks, 8.5 and 8.4 at the power limit).
template <class Matrix>
__device__ __forceinline__ void raised(Matrix matrix, int u) {
  __builtin_amdgcn_s_setprio(1);
  matrix(u);
  __builtin_amdgcn_s_setprio(0);
}
template <class Scores, class Matrix, class Vector, class Copy, class Wait>
__device__ __forceinline__ void alternate(int tiles, bool group_b, bool active, Scores scores, Matrix matrix, Vector vector,
                                          Copy copy, Wait wait) {
  if (group_b) {
    copy(0);
    wait(0);
  }
  __syncthreads();
  if (active) scores();
  if (active && !group_b) vector(0);
  __syncthreads();
  const int n = 2 * tiles;
  for (int u = 0; u < n; ++u) {
    if (!group_b) {
      if (active) raised(matrix, u);
    } else {
      if (u % 2 == 0 && u + 2 < n) copy(u / 2 + 1);
      if (active) vector(u);
    }
    __syncthreads();
    if (!group_b) {
      if (active && u + 1 < n) vector(u + 1);
    } else {
      if (active) raised(matrix, u);
      if (u % 2 == 0 && u + 2 < n) wait(u / 2 + 1);
    }
    __syncthreads();
  }
}

// dq.  A block: 8 waves of 32 queries, one per lane; K and V tiles of 64 keys double buffered in LDS.  S^T = K Q^T and
// dP^T = V dO^T leave a query's 16 keys in its lane, and dS^T is at once the operand of dQ^T += K^T dS^T.
// What bounds it: the parts of a step that the other group's matrix work does not cover, and power.  12 x 32760 x 32760 x 128 in
// bf16 takes 8.2 ms (1.2 PFLOP/s of three products) at 2.03 GHz with the matrix units busy in 56% of the cycles and LDS reading in
// 28%; on zeros, at 2.39 GHz, 7.2 and 55%.  fp16 8.8, 64 columns 5.5.  12 x 32760 x 512: 168 us.  Making delta here in place of
// its kernel cost 53 us there where that takes 61, whose loads come at the blocks' starts too: about 3% of the two, not taken.
template <int T, int DP, bool kFull>
__global__ void __launch_bounds__(kBwdWaves * kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
dense_dq_kernel(DenseArgs a) {
  constexpr int kAhead = 2, kS = DP / 16, kB = DP / 32, kElems = kBwdTile * DP;
  __shared__ __attribute__((aligned(16))) uint16_t k_s[2 * kElems], v_s[2 * kElems];
  __shared__ float scratch[2 * kBwdWaves];
  const unsigned total = (unsigned)a.batch * a.heads * a.tiles * a.splits, item = xcd_block(blockIdx.x, total);
  if (item >= total) return;
  const int tile = item % a.tiles, bh = item / a.tiles % (a.batch * a.heads), split = item / a.tiles / (a.batch * a.heads);
  const int b = bh / a.heads, head = bh % a.heads, kv = head / a.group;
  const int q_len = seq_len(a.q_lens, b, a.sq), k_len = seq_len(a.k_lens, b, a.sk);
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, h = lane / 32, l32 = lane % 32, wg = wave & 3;
  const int q0 = tile * kBwdRows, row = q0 + wave * 32 + l32;
  const int all = (k_len + kBwdTile - 1) / kBwdTile, per = (all + a.splits - 1) / a.splits;
  const int t0 = min(split * per, all), ntiles = q0 < q_len ? min(per, all - t0) : 0;
  const size_t to = (((size_t)b * a.sq + row) * a.heads + head) * a.d;
  f32x16_t acc[kB];
#pragma unroll
  for (int db = 0; db < kB; ++db) acc[db] = f32x16_t{};
  float e16 = 0.0f;
  if (ntiles > 0) {  // uniform
    start_apart<DP>(total, ntiles);
    if (T == kDenseF16) e16 = f16_exponent(a, b, kv, scratch);
    const float by = T == kDenseF16 ? __builtin_amdgcn_exp2f(e16) : 1.0f;
    const int r = min(row, q_len - 1);
    u32x4_t qop[kS], dop[kS];
    load_operand<DP, kFull>(a.q.p + (long long)b * a.q.batch + (long long)head * a.q.head + (long long)r * a.q.row, a.d, h, qop);
    load_operand<DP, kFull>(a.dy.p + (long long)b * a.dy.batch + (long long)head * a.dy.head + (long long)r * a.dy.row, a.d, h, dop);
    const float lse = a.lse[(size_t)bh * a.sq + r], nlse = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
    const float ndelta = -a.delta[(size_t)bh * a.sq + r] * by;
    const uint16_t* kb = a.k.p + (long long)b * a.k.batch + (long long)kv * a.k.head;
    const uint16_t* vb = a.v.p + (long long)b * a.v.batch + (long long)kv * a.v.head;
    TileReads<DP> at;
    at.init(lane);
    const int last = k_len - 1;
    if (!kFull) {
      tile_clear<DP, kBwdWaves * kWave, 2 * kElems>(k_s, a.d);
      tile_clear<DP, kBwdWaves * kWave, 2 * kElems>(v_s, a.d);
      __syncthreads();
    }
    f32x16_t s, dp;
    u32x4_t ds[2];
    auto place = [&](int u) __attribute__((always_inline)) { return u / 2 % 2 * kElems + u % 2 * 32 * DP; };
    auto copy = [&](int t) __attribute__((always_inline)) {
      tile_dma<DP, kFull, kBwdTile, 4>(kb, a.k.row, (t0 + t) * kBwdTile, last, a.d, k_s + t % 2 * kElems, wg, lane);
      tile_dma<DP, kFull, kBwdTile, 4>(vb, a.v.row, (t0 + t) * kBwdTile, last, a.d, v_s + t % 2 * kElems, wg, lane);
    };
    auto wait = [&](int) __attribute__((always_inline)) { __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
    // operands are read two instructions ahead
    auto products = [&](auto sums, const uint16_t* kt, const uint16_t* kn, const uint16_t* vn) __attribute__((always_inline)) {
      constexpr int kSums = decltype(sums)::value ? 2 * kB : 0, kAll = kSums + 2 * kS;
      u32x4_t op[kAhead + 1];
      auto operand = [&](int i) __attribute__((always_inline)) -> u32x4_t {
        if (i < kSums) return at.cols(kt + i / kB * 16 * DP, i % kB);
        return at.row((i - kSums) % 2 ? vn : kn, (i - kSums) / 2);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) op[i] = operand(i);
      if (kSums) __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
      else __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
      for (int i = 0; i < kAll; ++i) {
        if (i + kAhead < kAll) {
          op[(i + kAhead) % (kAhead + 1)] = operand(i + kAhead);
          if (i + kAhead < kSums) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        const int n = i - kSums;
        if (i < kSums) {
          acc[i % kB] = mma<T>(op[i % (kAhead + 1)], ds[i / kB], acc[i % kB]);
        } else if (n % 2 == 0) {
          if (n == 0) s = f32x16_t{};
          s = mma<T>(op[i % (kAhead + 1)], qop[n / 2], s);
        } else {
          if (n == 1) dp = f32x16_t{};
          dp = mma<T>(op[i % (kAhead + 1)], dop[n / 2], dp);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    };
    auto vector = [&](int u) __attribute__((always_inline)) {
      const int key0 = t0 * kBwdTile + u * 32;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, nlse)) *
               (T == kDenseF16 ? fmaf(dp[i], by, ndelta) : dp[i] + ndelta);
      }
      if (key0 + 32 > k_len) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + (i / 4) * 8 + h * 4 + (i % 4) >= k_len) s[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 16; i += 2) ds[i / 8][i % 8 / 2] = pack2<T>(s[i], s[i + 1]);
    };
    alternate(ntiles, wave >= 4, q0 + wave * 32 < q_len,
              [&]() __attribute__((always_inline)) { products(std::false_type(), k_s, k_s, v_s); },
              [&](int u) __attribute__((always_inline)) { products(std::true_type(), k_s + place(u), k_s + place(u + 1), v_s + place(u + 1)); },
              vector, copy, wait);
  }
  if (row >= a.sq) return;
  float by = row < q_len ? a.scale : 0.0f;
  if (T == kDenseF16) by *= __builtin_amdgcn_exp2f(-e16);
  if (row >= q_len)
#pragma unroll
    for (int db = 0; db < kB; ++db) acc[db] = f32x16_t{};
  if (a.splits > 1) {
#pragma unroll
    for (int db = 0; db < kB; ++db) acc[db] *= by;
    store_row32<DP, kFull>(a.part + (size_t)split * a.batch * a.sq * a.heads * a.d + to, acc, a.d, h);
  } else {
    store_row16<T, DP, kFull>(a.out + to, nullptr, acc, a.d, h, by);
  }
}

// dk, dv.  A block: 8 waves of 32 keys, one per lane; Q and dO tiles of 64 queries with their L and D double buffered in LDS.
// S = Q K^T and dP = dO V^T leave a key's 16 queries in its lane; P is at once the operand of dV^T += dO^T P, dS of
// dK^T += Q^T dS.  The two sums take 128 of a lane's 256 registers and K 32: V's operand is read from LDS where it is used
// (in registers too, they spill and 11.7 ms become 37).
// What bounds it: the same.  12 x 32760 x 32760 x 128 in bf16 takes 11.5 ms (1.15 PFLOP/s of four products) at 2.10 GHz with the
// matrix units busy in 52% of the cycles and LDS reading in 39%; on zeros, at 2.39 GHz, 10.2 and 52%.  fp16 12.5, 64 columns 7.8.
// 12 x 32760 x 512: 215 us, in shares of the queries.
template <int T, int DP, bool kFull>
__global__ void __launch_bounds__(kBwdWaves * kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
dense_dkv_kernel(DenseArgs a) {
  constexpr int kAhead = 2, kS = DP / 16, kB = DP / 32, kElems = kBwdTile * DP;
  __shared__ __attribute__((aligned(16))) uint16_t q_s[2 * kElems], d_s[2 * kElems], v_s[kBwdRows * DP];
  __shared__ __attribute__((aligned(16))) float stat_s[2][2][kBwdTile];  // -L log2(e) (fp16: + 14), -D
  __shared__ float scratch[2 * kBwdWaves];
  const unsigned total = (unsigned)a.batch * a.kv_heads * a.tiles * a.splits, item = xcd_block(blockIdx.x, total);
  if (item >= total) return;
  const int tile = item % a.tiles, bh = item / a.tiles % (a.batch * a.kv_heads), split = item / a.tiles / (a.batch * a.kv_heads);
  const int b = bh / a.kv_heads, kv = bh % a.kv_heads;
  const int q_len = seq_len(a.q_lens, b, a.sq), k_len = seq_len(a.k_lens, b, a.sk);
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, h = lane / 32, l32 = lane % 32, wg = wave & 3;
  const int k0 = tile * kBwdRows, row = k0 + wave * 32 + l32;
  const int qt = (q_len + kBwdTile - 1) / kBwdTile, all = qt * a.group, per = (all + a.splits - 1) / a.splits;
  const int t0 = min(split * per, all), ntiles = k0 < k_len ? min(per, all - t0) : 0;
  f32x16_t dk[kB], dv[kB];
#pragma unroll
  for (int db = 0; db < kB; ++db) dk[db] = dv[db] = f32x16_t{};
  float e16 = 0.0f;
  constexpr float kShift = T == kDenseF16 ? kF16PShift : 0.0f;
  if (ntiles > 0) {  // uniform
    if (T == kDenseF16) e16 = f16_exponent(a, b, kv, scratch);
    const float by = T == kDenseF16 ? __builtin_amdgcn_exp2f(e16 - kShift) : 1.0f;
    u32x4_t kop[kS];
    load_operand<DP, kFull>(a.k.p + (long long)b * a.k.batch + (long long)kv * a.k.head + (long long)min(row, k_len - 1) * a.k.row,
                            a.d, h, kop);
    TileReads<DP> at;
    at.init(lane);
    const int last = q_len - 1;
    if (!kFull) {
      tile_clear<DP, kBwdWaves * kWave, 2 * kElems>(q_s, a.d);
      tile_clear<DP, kBwdWaves * kWave, 2 * kElems>(d_s, a.d);
      tile_clear<DP, kBwdWaves * kWave, kBwdRows * DP>(v_s, a.d);
      __syncthreads();
    }
    tile_dma<DP, kFull, kBwdRows, kBwdWaves>(a.v.p + (long long)b * a.v.batch + (long long)kv * a.v.head, a.v.row, k0, k_len - 1,
                                             a.d, v_s, wave, lane);
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // published by the first barrier
    const uint16_t* vt = v_s + wave * 32 * DP;
    f32x16_t s, dp;
    u32x4_t p[2], ds[2];
    // L and D of a tile: group B's first 128 threads, a value each, loaded with the copies and left in LDS after them
    float stat = 0.0f;
    const int si = tid - 4 * kWave;
    int left = kBwdTile;  // queries from the copied tile's first on
    auto place = [&](int u) __attribute__((always_inline)) { return u / 2 % 2 * kElems + u % 2 * 32 * DP; };
    auto copy = [&](int t) __attribute__((always_inline)) {
      const int head = kv * a.group + (t0 + t) / qt, q0 = (t0 + t) % qt * kBwdTile;
      left = q_len - q0;
      tile_dma<DP, kFull, kBwdTile, 4>(a.q.p + (long long)b * a.q.batch + (long long)head * a.q.head, a.q.row, q0, last, a.d,
                                       q_s + t % 2 * kElems, wg, lane);
      tile_dma<DP, kFull, kBwdTile, 4>(a.dy.p + (long long)b * a.dy.batch + (long long)head * a.dy.head, a.dy.row, q0, last, a.d,
                                       d_s + t % 2 * kElems, wg, lane);
      if (si < 2 * kBwdTile) {
        const int q = q0 + si % kBwdTile;
        const size_t i = ((size_t)b * a.heads + head) * a.sq + min(q, last);
        stat = si < kBwdTile ? a.lse[i] : a.delta[i];
        if (q > last) stat = si < kBwdTile ? -INFINITY : 0.0f;
      }
    };
    auto wait = [&](int t) __attribute__((always_inline)) {
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (__builtin_expect(left < kBwdTile, 0)) tile_end<DP, kBwdTile, 4>(d_s + t % 2 * kElems, left, wg, lane);
      if (si < kBwdTile) stat_s[t % 2][0][si] = stat == -INFINITY ? -INFINITY : fmaf(-stat, kLog2e, kShift);
      else if (si < 2 * kBwdTile) stat_s[t % 2][1][si - kBwdTile] = -stat * by;
    };
    auto products = [&](auto sums, const uint16_t* qt_s, const uint16_t* dt_s, const uint16_t* qn, const uint16_t* dn)
                        __attribute__((always_inline)) {
      constexpr int kSums = decltype(sums)::value ? 4 * kB : 0, kAll = kSums + 2 * kS;
      u32x4_t op[kAhead + 1], vop[kAhead / 2 + 1];
      at.forget();
      auto operand = [&](int i) __attribute__((always_inline)) -> u32x4_t {
        if (i < kSums) return at.cols((i % 2 ? qt_s : dt_s) + i / 2 / kB * 16 * DP, i / 2 % kB);
        const int n = i - kSums;
        if (n % 2) vop[n / 2 % (kAhead / 2 + 1)] = at.row(vt, n / 2);
        return at.row(n % 2 ? dn : qn, n / 2);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) op[i] = operand(i);
      if (kSums) __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
      else __builtin_amdgcn_sched_group_barrier(0x100, kAhead + kAhead / 2, 0);
#pragma unroll
      for (int i = 0; i < kAll; ++i) {
        const int n = i - kSums;
        if (i + kAhead < kAll) {
          op[(i + kAhead) % (kAhead + 1)] = operand(i + kAhead);
          if (i + kAhead < kSums || (i + kAhead - kSums) % 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if (i < kSums) {
          const int db = i / 2 % kB, st = i / 2 / kB;
          if (i % 2) dk[db] = mma<T>(op[i % (kAhead + 1)], ds[st], dk[db]);
          else dv[db] = mma<T>(op[i % (kAhead + 1)], p[st], dv[db]);
        } else if (n % 2 == 0) {
          if (n == 0) s = f32x16_t{};
          s = mma<T>(op[i % (kAhead + 1)], kop[n / 2], s);
        } else {
          if (n == 1) dp = f32x16_t{};
          dp = mma<T>(op[i % (kAhead + 1)], vop[n / 2 % (kAhead / 2 + 1)], dp);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    };
    auto vector = [&](int u) __attribute__((always_inline)) {
      const float* st = &stat_s[u / 2 % 2][0][u % 2 * 32 + 4 * h];
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4_t nl = *(const f32x4_t*)(st + 8 * i4), nd = *(const f32x4_t*)(st + kBwdTile + 8 * i4);
        float pv[4], dv4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[e] = __builtin_amdgcn_exp2f(fmaf(s[4 * i4 + e], a.scale_log2, nl[e]));
          dv4[e] = pv[e] * (T == kDenseF16 ? fmaf(dp[4 * i4 + e], by, nd[e]) : dp[4 * i4 + e] + nd[e]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[i4 / 2][i4 % 2 * 2 + e] = pack2<T>(pv[2 * e], pv[2 * e + 1]);
          ds[i4 / 2][i4 % 2 * 2 + e] = pack2<T>(dv4[2 * e], dv4[2 * e + 1]);
        }
      }
    };
    alternate(ntiles, wave >= 4, k0 + wave * 32 < k_len,
              [&]() __attribute__((always_inline)) { products(std::false_type(), q_s, d_s, q_s, d_s); },
              [&](int u) __attribute__((always_inline)) {
                products(std::true_type(), q_s + place(u), d_s + place(u), q_s + place(u + 1), d_s + place(u + 1));
              },
              vector, copy, wait);
  }
  if (row >= a.sk) return;
  float byk = a.scale, byv = 1.0f;
  if (T == kDenseF16) {
    byk *= __builtin_amdgcn_exp2f(-e16);
    byv = __builtin_amdgcn_exp2f(-kShift);
  }
  if (row >= k_len)
#pragma unroll
    for (int db = 0; db < kB; ++db) dk[db] = dv[db] = f32x16_t{};
  const size_t to = (((size_t)b * a.sk + row) * a.kv_heads + kv) * a.d;
  if (a.splits > 1) {
    const size_t each = (size_t)a.batch * a.sk * a.kv_heads * a.d;
#pragma unroll
    for (int db = 0; db < kB; ++db) {
      dk[db] *= byk;
      dv[db] *= byv;
    }
    if (a.dk != nullptr) store_row32<DP, kFull>(a.part + split * each + to, dk, a.d, h);
    if (a.dv != nullptr) store_row32<DP, kFull>(a.part + (a.splits + split) * each + to, dv, a.d, h);
  } else {
    if (a.dk != nullptr) store_row16<T, DP, kFull>(a.dk + to, nullptr, dk, a.d, h, byk);
    if (a.dv != nullptr) store_row16<T, DP, kFull>(a.dv + to, nullptr, dv, a.d, h, byv);
  }
}

// Sums of the shares, four values a thread: of one result or two.
template <int T>
__global__ void __launch_bounds__(256) dense_sum_kernel(const float* part, size_t each, int splits, uint16_t* out0, uint16_t* out1) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  uint16_t* out = blockIdx.y == 0 ? out0 : out1;
  if (i >= each || out == nullptr) return;
  part += blockIdx.y * splits * each + i;
  f32x4_t v = *(const f32x4_t*)part;
  for (int s = 1; s < splits; ++s) v += *(const f32x4_t*)(part + s * each);
  *(uint2*)(out + i) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

struct BwdPlan {
  int q_splits, k_splits;
  size_t delta, norms, part, bytes;  // offsets, and the whole
};
static BwdPlan bwd_plan(int type, int batch, int heads, int kv_heads, int sq, int sk, int d, bool want_q, bool want_kv) {
  BwdPlan p = {};
  const long long qt = (sq + kBwdRows - 1) / kBwdRows, kt = (sk + kBwdRows - 1) / kBwdRows;
  const long long n_q = (long long)batch * sq * heads * d, n_k = (long long)batch * sk * kv_heads * d;
  p.q_splits = want_q ? dense_shares((long long)batch * heads * qt, (sk + kBwdTile - 1) / kBwdTile, n_q * 4) : 1;
  p.k_splits = want_kv ? dense_shares((long long)batch * kv_heads * kt, (long long)(heads / kv_heads) * ((sq + kBwdTile - 1) / kBwdTile), 2 * n_k * 4) : 1;
  auto take = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  p.delta = take((size_t)batch * heads * sq * sizeof(float));
  if (type == kDenseF16) p.norms = take(((size_t)batch * heads * qt + (size_t)batch * kv_heads * kt) * sizeof(float));
  // the two kernels' shares one after the other in the same place
  const size_t a = p.q_splits > 1 ? (size_t)p.q_splits * n_q * 4 : 0, c = p.k_splits > 1 ? (size_t)p.k_splits * 2 * n_k * 4 : 0;
  p.part = take(std::max(a, c));
  return p;
}

}  // namespace svoo

using namespace svoo;

extern "C" size_t svoo_dense_attention_bwd_workspace_size(int type, int batch, int heads, int kv_heads, int sq, int sk, int d,
                                                          int want_q, int want_kv) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || sq <= 0 || sk <= 0 || d <= 0) return 0;
  return bwd_plan(type, batch, heads, kv_heads, sq, sk, d, want_q != 0, want_kv != 0).bytes;
}

extern "C" int svoo_dense_attention_bwd(const void* dy, long long dy_batch, long long dy_head, long long dy_row, const void* q,
                                        long long q_batch, long long q_head, long long q_row, const void* k,
                                        long long k_batch, long long k_head, long long k_row, const void* v,
                                        long long v_batch, long long v_head, long long v_row, const void* o,
                                        long long o_batch, long long o_head, long long o_row, const void* o_rest,
                                        const float* lse, int type, int batch, int heads, int kv_heads, int sq, int sk, int d, float scale,
                                        const int32_t* q_lens, const int32_t* k_lens, void* dq, void* dk, void* dv,
                                        void* workspace, size_t ws_bytes, void* stream) {
  static const char* name = "svoo_dense_attention_bwd";
  if (const int rc = check_dense(name, type, batch, heads, kv_heads, sq, sk, d)) return rc;
  if (batch == 0 || heads == 0 || (sq == 0 && sk == 0) || (!dq && !dk && !dv)) return SVOO_OK;
  SVOO_REQUIRE(scale > 0.0f && scale < INFINITY, SVOO_ERR_INVALID_ARG, "%s: scale=%g", name, scale);
  SVOO_REQUIRE(sq > 0 && sk > 0, SVOO_ERR_INVALID_ARG, "%s: sq=%d sk=%d", name, sq, sk);
  SVOO_REQUIRE(dy && q && k && v && o && lse, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  DenseArgs a = {};
  a.dy = {(const uint16_t*)dy, dy_batch, dy_head, dy_row};
  a.q = {(const uint16_t*)q, q_batch, q_head, q_row};
  a.k = {(const uint16_t*)k, k_batch, k_head, k_row};
  a.v = {(const uint16_t*)v, v_batch, v_head, v_row};
  a.o = {(const uint16_t*)o, o_batch, o_head, o_row};
  SVOO_REQUIRE(dense_rows_ok(a.dy) && dense_rows_ok(a.q) && dense_rows_ok(a.k) && dense_rows_ok(a.v) && dense_rows_ok(a.o) &&
                   ((uintptr_t)o_rest | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0,
               SVOO_ERR_INVALID_ARG, "%s: rows at 16-byte addresses", name);
  const BwdPlan p = bwd_plan(type, batch, heads, kv_heads, sq, sk, d, dq != nullptr, dk || dv);
  SVOO_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && ws_bytes >= p.bytes, SVOO_ERR_WORKSPACE,
               "%s: workspace of %zu bytes (%zu needed)", name, ws_bytes, p.bytes);
  char* ws = (char*)workspace;
  a.rest = (uint16_t*)o_rest;
  a.lse = (float*)lse;
  a.delta = (float*)(ws + p.delta);
  a.norms = (float*)(ws + p.norms);
  a.part = (float*)(ws + p.part);
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.batch = batch;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.sq = sq;
  a.sk = sk;
  a.d = d;
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  hipStream_t s = (hipStream_t)stream;
  const int q_tiles = (sq + kBwdRows - 1) / kBwdRows, k_tiles = (sk + kBwdRows - 1) / kBwdRows;
  const int q_blocks = batch * heads * q_tiles, v_blocks = type == kDenseF16 ? batch * kv_heads * k_tiles : 0;
  for_dense(type, d, [&](auto type_tag, auto dp_tag, auto full_tag) {
    constexpr int kT = decltype(type_tag)::value, kDP = decltype(dp_tag)::value;
    constexpr bool kFull = decltype(full_tag)::value;
    static_assert(kNormRows == kBwdRows, "a maximum for every block of rows");
    hipLaunchKernelGGL((dense_delta_kernel<kT>), dim3((unsigned)(q_blocks + v_blocks)), dim3(kDeltaThreads), 0, s, a, q_blocks, v_blocks);
    const dim3 block(kBwdWaves * kWave);
    auto sum = [&](size_t each, int splits, void* out0, void* out1) {
      hipLaunchKernelGGL((dense_sum_kernel<kT>), dim3((unsigned)((each / 4 + 255) / 256), out1 ? 2 : 1), dim3(256), 0, s, a.part,
                         each, splits, (uint16_t*)out0, (uint16_t*)out1);
    };
    if (dq) {
      a.out = (uint16_t*)dq;
      a.tiles = q_tiles;
      a.splits = p.q_splits;
      const unsigned total = (unsigned)q_blocks * a.splits;
      hipLaunchKernelGGL((dense_dq_kernel<kT, kDP, kFull>), dim3((total + 7) / 8 * 8), block, 0, s, a);
      if (a.splits > 1) sum((size_t)batch * sq * heads * d, a.splits, dq, nullptr);
    }
    if (dk || dv) {
      a.dk = (uint16_t*)dk;
      a.dv = (uint16_t*)dv;
      a.tiles = k_tiles;
      a.splits = p.k_splits;
      const unsigned total = (unsigned)batch * kv_heads * k_tiles * a.splits;
      hipLaunchKernelGGL((dense_dkv_kernel<kT, kDP, kFull>), dim3((total + 7) / 8 * 8), block, 0, s, a);
      if (a.splits > 1) sum((size_t)batch * sk * kv_heads * d, a.splits, dk, dv);
    }
  });
  return check_launch(name);
}
