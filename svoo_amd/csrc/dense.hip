// Dense attention: the forward pass, the C entries.
#include "dense.h"

namespace svoo {

constexpr int kFwdWaves = 8, kFwdQ = kFwdWaves * 32, kFwdK = 64;

// A block: 8 waves of 32 queries.  K and V tiles of 64 keys are double buffered in LDS and filled by LDS DMA.  The two waves
// of a SIMD belong to two groups that alternate, half a step apart, between a tile's matrix work {O += V(t)^T P(t)^T,
// S(t+1) = K(t+1) Q^T} and the softmax of the next, so that matrix and vector units are busy at the same time.
//
// What bounds it: how much of the softmax and the barriers the other group's matrix work covers, and the chip's power.  12 heads
// of 32760 x 32760, 128 columns, bf16, take 5.5 ms (1.2 PFLOP/s) at 1.97 GHz, matrix units busy in 58% of the cycles, LDS reading
// in 29% without bank conflicts; on zeros, at 2.39 GHz, 4.5 ms and 56%.  fp16 6.1 ms.  64 columns 3.64 ms, matrix units busy in
// 37%, LDS in 28%, 9% bank conflicts of the transposing reads.  12 x 32760 x 512: 130 us (0.8 PFLOP/s), a third of it the ends
// of so short a walk; one query over 12 x 32760 keys: 38 us (5.3 TB/s).  Blocks of four waves, two of them on a CU, overlap
// these ends but read K and V twice as often: 142 and 148 us with 512 keys, 6.3 ms with 32760.  Walking over several query
// tiles in one block spills (7.7 ms, and 6.8 with chains of tiles).
template <int T, int DP, bool kFull>
__global__ void __launch_bounds__(kFwdWaves * kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
dense_fwd_kernel(DenseArgs a) {
  constexpr int kS = DP / 16, kB = DP / 32;
  __shared__ __attribute__((aligned(16))) uint16_t k_s[2][kFwdK * DP], v_s[2][kFwdK * DP];
  const unsigned total = (unsigned)a.batch * a.heads * a.tiles * a.splits, item = xcd_block(blockIdx.x, total);
  if (item >= total) return;
  // split outermost, then head, then tile
  const int tile = item % a.tiles, bh = item / a.tiles % (a.batch * a.heads), split = item / a.tiles / (a.batch * a.heads);
  const int b = bh / a.heads, head = bh % a.heads, kv = head / a.group;
  const int q_len = seq_len(a.q_lens, b, a.sq), k_len = seq_len(a.k_lens, b, a.sk);
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, h = lane / 32, l32 = lane % 32, wg = wave & 3;
  const bool group_b = wave >= 4;
  const int q0 = tile * kFwdQ, row = q0 + wave * 32 + l32;
  // this share's keys, whole tiles
  const int all = (k_len + kFwdK - 1) / kFwdK, per = (all + a.splits - 1) / a.splits;
  const int t0 = min(split * per, all), ntiles = min(per, all - t0);
  const size_t stat = (size_t)bh * a.sq;
  const size_t out0 = ((size_t)b * a.sq * a.heads + head) * a.d;
  auto zero_row = [&]() __attribute__((always_inline)) {
    const size_t to = out0 + (size_t)row * a.heads * a.d;
    for (int c = 4 * h; c < a.d; c += 8) {
      *(uint2*)(a.out + to + c) = make_uint2(0, 0);
      if (a.rest != nullptr) *(uint2*)(a.rest + to + c) = make_uint2(0, 0);
    }
    if (h == 0) a.lse[stat + row] = -INFINITY;
  };
  if (ntiles <= 0 || q0 >= q_len) {  // no keys, or padding only
    if (row < a.sq) {
      if (a.splits > 1) {
        if (h == 0) a.part_ml[(size_t)split * a.batch * a.heads * a.sq + stat + row] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
      } else {
        zero_row();
      }
    }
    return;
  }
  const bool active = q0 + wave * 32 < q_len;  // uniform over the wave
  start_apart<DP>(total, ntiles);
  u32x4_t qop[kS];
  load_operand<DP, kFull>(a.q.p + (long long)b * a.q.batch + (long long)head * a.q.head + (long long)min(row, q_len - 1) * a.q.row, a.d,
                   h, qop);
  const uint16_t* kb = a.k.p + (long long)b * a.k.batch + (long long)kv * a.k.head;
  const uint16_t* vb = a.v.p + (long long)b * a.v.batch + (long long)kv * a.v.head;
  TileReads<DP> at;
  at.init(lane);
  f32x16_t acc[kB], sacc[2];
#pragma unroll
  for (int db = 0; db < kB; ++db) acc[db] = f32x16_t{};
  float m_run = kLowest, l_run = 0.0f, w_run = 0.0f;  // the maximum, the sum of P, and the sum of P as it multiplies V
  u32x4_t pop[2][2];
  const float sl = a.scale_log2;
  const int last = k_len - 1;
  auto dma = [&](const DenseRows& m, const uint16_t* base, int t, uint16_t* to) __attribute__((always_inline)) {
    tile_dma<DP, kFull, kFwdK, 4>(base, m.row, (t0 + t) * kFwdK, last, a.d, to, wg, lane);
  };
  // the copied V(t) is there, its rows behind the last key zeros
  const int ragged = k_len % kFwdK != 0 ? all - 1 - t0 : -1;  // the tile with such rows
  auto v_there = [&](int t, uint16_t* tile) __attribute__((always_inline)) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (__builtin_expect(t == ragged, 0)) tile_end<DP, kFwdK, 4>(tile, k_len % kFwdK, wg, lane);
  };
  auto scores = [&](const uint16_t* kt) __attribute__((always_inline)) {
    sacc[0] = f32x16_t{};
    sacc[1] = f32x16_t{};
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2)
        sacc[kb2] = mma<T>(at.row(kt + kb2 * 32 * DP, s), qop[s], sacc[kb2]);
  };
  // O += V(t)^T P(t)^T, then S(t+1): one pipeline whose operand reads run two instructions ahead
  constexpr int kPv = 4 * kB, kAll = kPv + 2 * kS;
  auto operand = [&](int i, const uint16_t* vt, const uint16_t* kn) __attribute__((always_inline)) -> u32x4_t {
    if (i < kPv) {
      const int rb = (i / kB) * 16 * DP, db = i % kB;
      return at.cols(vt + rb, db);
    }
    const int j = i - kPv;
    return at.row(kn + (j % 2) * 32 * DP, j / 2);
  };
  auto mphase = [&](const uint16_t* vt, const uint16_t* kn) __attribute__((always_inline)) {
    u32x4_t buf[3];
    buf[0] = operand(0, vt, kn);
    buf[1] = operand(1, vt, kn);
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
      if (i + 2 < kAll) {
        buf[(i + 2) % 3] = operand(i + 2, vt, kn);
        if (i + 2 < kPv) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      if (i < kPv) {
        const int kb2 = i / kB / 2, st = i / kB % 2, db = i % kB;
        acc[db] = mma<T>(buf[i % 3], pop[kb2][st], acc[db]);
      } else {
        const int j = i - kPv;
        if (j < 2) sacc[j] = f32x16_t{};
        sacc[j % 2] = mma<T>(buf[i % 3], qop[j / 2], sacc[j % 2]);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
  };
  // softmax of S(t).  bf16: against a running maximum that moves only when the lane's sum of 32 leaves [0, 2^13].  fp16: against
  // 2^-kF16Top of one that moves only when a score would take P out of the type; finding the tile's highest score first costs
  // 2.5 to 5% (12 x 32760 x 32760: 128 columns 6.10 ms of 5.93, 64 columns 4.16 of 3.98), where asking the packed P for
  // infinities costs 2 to 7 (scores of deviation 1 and 4) and, over 512 keys of deviation 2, 20 (166 us; 148 so, 137 without).
  auto vphase = [&](int t) __attribute__((always_inline)) {
    if ((t0 + t + 1) * kFwdK > k_len) {
      const int base = (t0 + t) * kFwdK;
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (base + kb2 * 32 + (r / 4) * 8 + h * 4 + (r % 4) >= k_len) sacc[kb2][r] = -INFINITY;
    }
    float wsum;
    auto pexp = [&]() __attribute__((always_inline)) -> float {
      float la[4] = {0.0f, 0.0f, 0.0f, 0.0f}, wa[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2) {
        float pv[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) pv[r] = __builtin_amdgcn_exp2f(fmaf(sacc[kb2][r], sl, -m_run));
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int e = 0; e < 4; ++e) pop[kb2][st][e] = pack2<T>(pv[8 * st + 2 * e], pv[8 * st + 2 * e + 1]);
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int e = 0; e < 4; ++e) wa[e] = sum2<T>(pop[kb2][st][e], wa[e]);
#pragma unroll
        for (int r = 0; r < 16; ++r) la[r % 4] += pv[r];
      }
      wsum = (wa[0] + wa[1]) + (wa[2] + wa[3]);
      return (la[0] + la[1]) + (la[2] + la[3]);
    };
    auto highest = [&]() __attribute__((always_inline)) -> float {
      float mx = sacc[0][0];
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kb2][r]);
      return mx;
    };
    auto move = [&](bool high, float mx) __attribute__((always_inline)) {
      mx = xhalf_max(mx) * sl;
      // a row's maximum moves for its own sake alone: its bits do not depend on the rows beside it
      const bool moves = xhalf_max(high ? 1.0f : 0.0f) > 0.0f;
      const float low = T == kDenseF16 && fabsf(mx) < kF16TopWithin ? mx - kF16Top : mx;
      const float m_new = moves ? fmaxf(m_run, low) : m_run;
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      w_run *= alpha;
#pragma unroll
      for (int db = 0; db < kB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
    };
    float lsum;
    if (T == kDenseF16) {
      const float mx = highest();
      const bool high = fmaf(mx, sl, -m_run) > 15.9f;
      if (__any(high)) move(high, mx);
      lsum = pexp();
    } else {
      lsum = pexp();
      const bool high = !(lsum <= 8192.0f);
      if (__any(high)) {
        move(high, highest());
        lsum = pexp();
      }
    }
    l_run += lsum;
    w_run += wsum;
  };
  if (!kFull) {
    tile_clear<DP, kFwdWaves * kWave, 2 * kFwdK * DP>(k_s[0], a.d);
    tile_clear<DP, kFwdWaves * kWave, 2 * kFwdK * DP>(v_s[0], a.d);
    __syncthreads();
  }
  // Prologue: K(0), V(0), K(1); S(0) everywhere, P(0) in group A.
  if (group_b) {
    dma(a.k, kb, 0, k_s[0]);
    dma(a.v, vb, 0, v_s[0]);
    dma(a.k, kb, 1, k_s[1]);
    v_there(0, v_s[0]);
  }
  __syncthreads();
  if (active) scores(k_s[0]);
  if (active && !group_b) vphase(0);
  __syncthreads();
  // Half-steps.  A: M(t), then P(t+1).  B: P(t) with the copies of K(t+2) and V(t+1), then M(t).  Copies of tiles behind the
  // end read the last row again, and S behind the last tile is not used.
  for (int t = 0; t < ntiles; t += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (t + u < ntiles) {
        if (!group_b) {
          if (active) mphase(v_s[u], k_s[u ^ 1]);
        } else {
          dma(a.k, kb, t + u + 2, k_s[u]);
          dma(a.v, vb, t + u + 1, v_s[u ^ 1]);
          if (active) vphase(t + u);
        }
        __syncthreads();
        if (!group_b) {
          if (active && t + u + 1 < ntiles) vphase(t + u + 1);
        } else {
          if (active) mphase(v_s[u], k_s[u ^ 1]);
          v_there(t + u + 1, v_s[u ^ 1]);
        }
        __syncthreads();
      }
    }
  }
  l_run = xhalf_sum(l_run);
  w_run = xhalf_sum(w_run);
  if (row >= a.sq) return;
  if (a.splits > 1) {
    const size_t to = (size_t)split * a.batch * a.heads * a.sq + stat + row;
    if (h == 0) a.part_ml[to] = row < q_len ? make_float4(m_run, l_run, w_run, 0.0f) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    store_row32<DP, kFull>(a.part + to * a.d, acc, a.d, h);
    return;
  }
  if (row < q_len) {
    const size_t to = out0 + (size_t)row * a.heads * a.d;
    store_row16<T, DP, kFull>(a.out + to, a.rest != nullptr ? a.rest + to : nullptr, acc, a.d, h, 1.0f / w_run);
    if (h == 0) a.lse[stat + row] = row_lse(m_run, l_run);
  } else {
    zero_row();
  }
}

// Joins the shares of a query's keys.  A thread takes four columns and every kJoinSlices-th share, and these meet in LDS.
// Memory's latency bounds it.  Eight slices and one: 5 and 15 us for 128 shares of 12 rows, 12.0 and 17.8 for 21 shares of
// 12 x 256 rows, 13.9 and 11.2 for ten of 12 x 512, 30 and 9.4 for two of 24888.
template <int T, int kJoinSlices>
__global__ void __launch_bounds__(256) dense_join_kernel(DenseArgs a) {
  __shared__ f32x4_t s_o[256];
  __shared__ float s_m[256], s_l[256], s_w[256];
  const int per_row = a.d / 4, here = 256 / (per_row * kJoinSlices);  // rows of a block
  const int c = threadIdx.x % per_row, slice = threadIdx.x / per_row % kJoinSlices, mine = threadIdx.x / (per_row * kJoinSlices);
  const size_t rows = (size_t)a.batch * a.heads * a.sq, at = (size_t)blockIdx.x * here + mine;
  const bool on = mine < here && at < rows;
  float m = -INFINITY, l = 0.0f, lw = 0.0f;
  f32x4_t o = {0, 0, 0, 0};
  if (on) {
    for (int s = slice; s < a.splits; s += kJoinSlices) m = fmaxf(m, a.part_ml[s * rows + at].x);
#pragma unroll 4
    for (int s = slice; s < a.splits; s += kJoinSlices) {
      const float4 ml = a.part_ml[s * rows + at];
      if (ml.x == -INFINITY) continue;  // an empty share wrote no row
      const float w = __builtin_amdgcn_exp2f(ml.x - m);
      l = fmaf(ml.y, w, l);
      lw = fmaf(ml.z, w, lw);
      o += *(const f32x4_t*)(a.part + (s * rows + at) * a.d + 4 * c) * w;
    }
  }
  s_o[threadIdx.x] = o;
  s_m[threadIdx.x] = m;
  s_l[threadIdx.x] = l;
  s_w[threadIdx.x] = lw;
  __syncthreads();
  if (!on || slice != 0) return;
#pragma unroll
  for (int i = 1; i < kJoinSlices; ++i) m = fmaxf(m, s_m[threadIdx.x + i * per_row]);
  o = f32x4_t{0, 0, 0, 0};
  l = lw = 0.0f;
#pragma unroll
  for (int i = 0; i < kJoinSlices; ++i) {
    const int j = threadIdx.x + i * per_row;
    if (s_m[j] == -INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(s_m[j] - m);
    l = fmaf(s_l[j], w, l);
    lw = fmaf(s_w[j], w, lw);
    o += s_o[j] * w;
  }
  const bool some = m > -INFINITY;  // keys: the lowest maximum of a share with any is kLowest
  const int row = (int)(at % a.sq), bh = (int)(at / a.sq);
  const size_t to = ((size_t)(bh / a.heads) * a.sq + row) * a.heads * a.d + (size_t)(bh % a.heads) * a.d + 4 * c;
  o *= some ? 1.0f / lw : 0.0f;
  const uint2 w = pack4<T>(o);
  *(uint2*)(a.out + to) = w;
  if (a.rest != nullptr) *(uint2*)(a.rest + to) = pack4<T>(rest4<T>(o, w));
  if (c == 0) a.lse[at] = some ? row_lse(m, l) : -INFINITY;
}

// Shares of the contracted length for a launch of `blocks` blocks that each walk over `units` tiles: the fewest rounds of 256
// resident blocks times tiles, with two tiles' time for writing and joining partial results.  With shares and in one: a query
// over 12 x 32760 keys 43 and 577 us; dk and dv of 12 x 512 keys from 32760 queries 260 and 1750, of 3 x 2 x 771 keys from 4
// heads of 1037 queries 36 and 181; nothing to win with 12 x 128 blocks (two shares 145 us, one 154).
int dense_shares(long long blocks, long long units, long long bytes) {
  long long best = 1, cost = (blocks + 255) / 256 * units;
  for (long long s = 2; s <= 256 && s * 4 <= units && s * bytes <= (256ll << 20); ++s) {
    const long long c = (blocks * s + 255) / 256 * ((units + s - 1) / s + 2) + 2;
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return (int)best;
}
static long long fwd_blocks(int batch, int heads, int sq) { return (long long)batch * heads * ((sq + kFwdQ - 1) / kFwdQ); }

static int fwd_splits(int batch, int heads, int sq, int sk, int d) {
  return dense_shares(fwd_blocks(batch, heads, sq), (sk + kFwdK - 1) / kFwdK, (long long)batch * heads * sq * d * 4);
}

bool dense_rows_ok(const DenseRows& m) {
  return (uintptr_t)m.p % 16 == 0 && m.batch % 8 == 0 && m.head % 8 == 0 && m.row % 8 == 0 && m.row >= 0 && m.row < (1 << 23);
}
int check_dense(const char* name, int type, int batch, int heads, int kv_heads, int sq, int sk, int d) {
  SVOO_REQUIRE(type == kDenseBf16 || type == kDenseF16, SVOO_ERR_INVALID_ARG, "%s: element type %d (0 bf16, 1 fp16)", name, type);
  SVOO_REQUIRE(batch >= 0 && heads >= 0 && kv_heads >= 0 && sq >= 0 && sk >= 0 && d > 0, SVOO_ERR_INVALID_ARG,
               "%s: batch=%d heads=%d, %d sq=%d sk=%d d=%d", name, batch, heads, kv_heads, sq, sk, d);
  SVOO_REQUIRE(d <= 128 && d % 8 == 0, SVOO_ERR_UNSUPPORTED, "%s: d=%d (multiples of 8 up to 128)", name, d);
  SVOO_REQUIRE(heads == 0 || (kv_heads > 0 && heads % kv_heads == 0), SVOO_ERR_INVALID_ARG, "%s: %d heads share %d", name, heads,
               kv_heads);
  SVOO_REQUIRE(sq <= (1 << 30) && sk <= (1 << 30), SVOO_ERR_UNSUPPORTED, "%s: sq=%d sk=%d (up to 2^30)", name, sq, sk);
  // fewer than 2^32 threads in a launch, also with 512 blocks' worth of shares
  SVOO_REQUIRE(fwd_blocks(batch, heads, sq) < (1ll << 22) && fwd_blocks(batch, heads, sk) < (1ll << 22), SVOO_ERR_UNSUPPORTED,
               "%s: %d x %d heads of %d queries and %d keys (2^22 tiles of 256 rows or more)", name, batch, heads, sq, sk);
  return SVOO_OK;
}

}  // namespace svoo

using namespace svoo;

extern "C" size_t svoo_dense_attention_fwd_workspace_size(int batch, int heads, int sq, int sk, int d) {
  if (batch <= 0 || heads <= 0 || sq <= 0 || sk <= 0 || d <= 0) return 0;
  const int splits = fwd_splits(batch, heads, sq, sk, d);
  return splits == 1 ? 0 : (size_t)splits * batch * heads * sq * (d * sizeof(float) + sizeof(float4));
}

extern "C" int svoo_dense_attention_fwd(const void* q, long long q_batch, long long q_head, long long q_row, const void* k,
                                        long long k_batch, long long k_head, long long k_row, const void* v,
                                        long long v_batch, long long v_head, long long v_row, int type, int batch, int heads,
                                        int kv_heads, int sq, int sk, int d, float scale, const int32_t* q_lens,
                                        const int32_t* k_lens, void* o, void* o_rest, float* lse, void* workspace,
                                        size_t ws_bytes, void* stream) {
  static const char* name = "svoo_dense_attention_fwd";
  if (const int rc = check_dense(name, type, batch, heads, kv_heads, sq, sk, d)) return rc;
  if (batch == 0 || heads == 0 || sq == 0) return SVOO_OK;
  SVOO_REQUIRE(scale > 0.0f && scale < INFINITY, SVOO_ERR_INVALID_ARG, "%s: scale=%g", name, scale);
  SVOO_REQUIRE(q && (sk == 0 || (k && v)) && o && lse, SVOO_ERR_INVALID_ARG, "%s: null pointer", name);
  DenseArgs a = {};
  a.q = {(const uint16_t*)q, q_batch, q_head, q_row};
  a.k = {(const uint16_t*)k, k_batch, k_head, k_row};
  a.v = {(const uint16_t*)v, v_batch, v_head, v_row};
  SVOO_REQUIRE(dense_rows_ok(a.q) && dense_rows_ok(a.k) && dense_rows_ok(a.v) && ((uintptr_t)o | (uintptr_t)o_rest) % 16 == 0, SVOO_ERR_INVALID_ARG,
               "%s: rows at 16-byte addresses", name);
  a.out = (uint16_t*)o;
  a.rest = (uint16_t*)o_rest;
  a.lse = lse;
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
  a.tiles = (sq + kFwdQ - 1) / kFwdQ;
  a.splits = fwd_splits(batch, heads, sq, sk, d);
  const size_t need = svoo_dense_attention_fwd_workspace_size(batch, heads, sq, sk, d);
  SVOO_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && ws_bytes >= need), SVOO_ERR_WORKSPACE, "%s: workspace of %zu bytes (%zu needed)", name,
               ws_bytes, need);
  const size_t rows = (size_t)batch * heads * sq;
  a.part = (float*)workspace;
  a.part_ml = (float4*)((float*)workspace + (need ? (size_t)a.splits * rows * d : 0));
  const unsigned total = (unsigned)batch * heads * a.tiles * a.splits;
  const dim3 grid((total + 7) / 8 * 8), block(kFwdWaves * kWave);
  for_dense(type, d, [&](auto t, auto dp, auto full) {
    constexpr int kT = decltype(t)::value;
    hipLaunchKernelGGL((dense_fwd_kernel<kT, decltype(dp)::value, decltype(full)::value>), grid, block, 0, (hipStream_t)stream, a);
    auto join = [&](auto slices) {
      constexpr int kSlices = decltype(slices)::value;
      const size_t here = 256 / (d / 4 * kSlices);
      hipLaunchKernelGGL((dense_join_kernel<kT, kSlices>), dim3((unsigned)((rows + here - 1) / here)), dim3(256), 0,
                         (hipStream_t)stream, a);
    };
    if (a.splits > 16) join(std::integral_constant<int, 8>());
    else if (a.splits > 1) join(std::integral_constant<int, 1>());
  });
  return check_launch(name);
}
