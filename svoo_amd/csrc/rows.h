// Eight consecutive elements of a row per lane, whatever the element type and the row's address; sums and maxima over
// the lanes of a row; 8-bit values with a power-of-two scale per block of 128.
#pragma once

#include "svoo_common.h"

namespace svoo {

enum RowType { kRowBf16 = 0, kRowF16 = 1, kRowF32 = 2 };
enum Fp8Type { kFp8E4m3 = 0, kFp8E5m2 = 1 };

// Four dwords at any byte address (gfx950's global loads and stores need no alignment).
struct __attribute__((packed, aligned(1))) Dwords4 { u32x4_t v; };
struct __attribute__((packed, aligned(1))) Dwords2 { uint32_t v[2]; };
struct __attribute__((packed, aligned(1))) Dword { uint32_t v; };

__device__ __forceinline__ float row_elem(const void* p, int type, long long i) {
  if (type == kRowBf16) return bf16_to_f32(((const uint16_t*)p)[i]);
  if (type == kRowF16) return (float)__builtin_bit_cast(_Float16, ((const uint16_t*)p)[i]);
  return ((const float*)p)[i];
}

__device__ __forceinline__ void set_row_elem(void* p, int type, long long i, float v) {
  if (type == kRowBf16) ((uint16_t*)p)[i] = f32_to_bf16(v);
  else if (type == kRowF16) ((uint16_t*)p)[i] = __builtin_bit_cast(uint16_t, (_Float16)v);
  else ((float*)p)[i] = v;
}

// v as the row's type holds it.
template <int T>
__device__ __forceinline__ void round_row8(float (&f)[8]) {  // to the type and back
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    if (T == kRowBf16) {
      const uint32_t w = cvt_pk_bf16(f[e], f[e + 1]);
      f[e] = __uint_as_float(w << 16);
      f[e + 1] = __uint_as_float(w & 0xffff0000u);
    } else if (T == kRowF16) {
      f[e] = (float)(_Float16)f[e];
      f[e + 1] = (float)(_Float16)f[e + 1];
    }
  }
}

// Elements i .. i + 7 of a row, the first n of them (n <= 0: none) and zeros.  kWhole: n is a multiple of 8.
template <int T, bool kWhole = false>
__device__ __forceinline__ void load_row8(const void* p, long long i, int n, float (&f)[8]) {
  if (n >= 8) {
    if (T == kRowF32) {
      const u32x4_t a = ((const Dwords4*)((const float*)p + i))->v, b = ((const Dwords4*)((const float*)p + i + 4))->v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = __uint_as_float(a[e]);
        f[4 + e] = __uint_as_float(b[e]);
      }
    } else {
      const u32x4_t w = ((const Dwords4*)((const uint16_t*)p + i))->v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t b = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
        f[e] = T == kRowBf16 ? bf16_to_f32(b) : (float)__builtin_bit_cast(_Float16, b);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = !kWhole && e < n ? row_elem(p, T, i + e) : 0.0f;
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

template <int T, bool kWhole = false>
__device__ __forceinline__ void store_row8(void* p, long long i, int n, const float (&f)[8]) {
  if (T == kRowF32) {
    float* to = (float*)p + i;
    const u32x4_t a = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    const u32x4_t b = {__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
    if (n >= 8) {
      ((Dwords4*)to)->v = a;
      ((Dwords4*)(to + 4))->v = b;
    } else if (!kWhole && n > 0) {
      if (n & 4) ((Dwords4*)to)->v = a;
      const u32x4_t rest = n & 4 ? b : a;
      to += n & 4;
      if (n & 2) *(Dwords2*)to = Dwords2{{rest[0], rest[1]}};
      if (n & 1) *(Dword*)(to + (n & 2)) = Dword{n & 2 ? rest[2] : rest[0]};
    }
  } else {
    u32x4_t w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (T == kRowBf16) {
        w[e] = cvt_pk_bf16(f[2 * e], f[2 * e + 1]);
      } else {
        w[e] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * e]) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * e + 1]) << 16);
      }
    }
    if (n >= 8) ((Dwords4*)((uint16_t*)p + i))->v = w;
    else if (!kWhole) store_row8_bits((uint16_t*)p + i, n, w);
  }
}

// A row's share of lane t of TPR as it lies in memory: NC chunks of eight elements, (c TPR + t) 8 .. + 7 of cols, zeros
// past the end.  Half as many registers as its values in fp32 take; they are converted where they are used.
template <int T, int NC>
struct RawRow {
  u32x4_t v[NC][T == kRowF32 ? 2 : 1];

  template <int TPR, bool kWhole>
  __device__ __forceinline__ void load(const void* p, long long at, int cols, int t) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int n = cols - (c * TPR + t) * 8;
      const long long i = at + (c * TPR + t) * 8;
      if (n >= 8) {
        if (T == kRowF32) {
          v[c][0] = ((const Dwords4*)((const float*)p + i))->v;
          v[c][T == kRowF32 ? 1 : 0] = ((const Dwords4*)((const float*)p + i + 4))->v;
        } else {
          v[c][0] = ((const Dwords4*)((const uint16_t*)p + i))->v;
        }
      } else {
#pragma unroll
        for (int h = 0; h < (T == kRowF32 ? 2 : 1); ++h) v[c][h] = u32x4_t{0, 0, 0, 0};
        if (!kWhole && TPR > 16) {  // more than eight columns: the last eight, moved down
          if (n > 0) load_end(v[c], p, i + n - 8, 8 - n);
        } else if (!kWhole) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) {
              if (T == kRowF32) v[c][T == kRowF32 ? e / 4 : 0][e % 4] = ((const uint32_t*)p)[i + e];
              else v[c][0][e / 2] |= (uint32_t)((const uint16_t*)p)[i + e] << (16 * (e & 1));
            }
        }
      }
    }
  }
  // Elements i + by .. i + 7 to the front, zeros behind; by is 1 to 7.
  static __device__ __forceinline__ void load_end(u32x4_t (&to)[T == kRowF32 ? 2 : 1], const void* p, long long i, int by) {
    if (T == kRowF32) {
      const u32x4_t a = ((const Dwords4*)((const float*)p + i))->v, b = ((const Dwords4*)((const float*)p + i + 4))->v;
      uint32_t w[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
      for (int step = 4; step > 0; step /= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = by & step ? (e + step < 8 ? w[e + step < 8 ? e + step : 0] : 0u) : w[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) to[T == kRowF32 ? e / 4 : 0][e % 4] = w[e];
    } else {
      const u32x4_t a = ((const Dwords4*)((const uint16_t*)p + i))->v;
      unsigned long long lo = a[0] | (unsigned long long)a[1] << 32, hi = a[2] | (unsigned long long)a[3] << 32;
      if (by >= 4) {
        lo = hi;
        hi = 0;
      }
      const int bits = by % 4 * 16;
      lo = lo >> bits | (bits ? hi << (64 - bits) : 0ull);
      hi >>= bits;
      to[0] = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
  }
  // Values converted before are converted again: held in fp32 they would take the registers that this type saves.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int h = 0; h < (T == kRowF32 ? 2 : 1); ++h) __asm__ volatile("" : "+v"(v[c][h]));
  }
  __device__ __forceinline__ float at(int c, int e) const {
    if (T == kRowF32) return __uint_as_float(v[c][T == kRowF32 ? e / 4 : 0][e % 4]);
    if (T == kRowBf16) return __uint_as_float(e & 1 ? v[c][0][e / 2] & 0xffff0000u : v[c][0][e / 2] << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[c][0][e / 2] >> (16 * (e & 1))));
  }
};

// Eight values of a row's share to memory, by the (uniform) type.
template <bool kWhole>
__device__ __forceinline__ void store_row8_as(void* p, int type, long long i, int n, const float (&f)[8]) {
  if (type == kRowBf16) store_row8<kRowBf16, kWhole>(p, i, n, f);
  else if (type == kRowF16) store_row8<kRowF16, kWhole>(p, i, n, f);
  else store_row8<kRowF32, kWhole>(p, i, n, f);
}

// ---------------------------------------------------------------- sums and maxima over lanes, in every lane
template <int N>
__device__ __forceinline__ float rotated16(float v) {  // lane i of 16 sees lane (i - N) % 16
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float sum16(float v) {
  v += rotated16<8>(v);
  v += rotated16<4>(v);
  v += rotated16<2>(v);
  return v + rotated16<1>(v);
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, rotated16<8>(v));
  v = fmaxf(v, rotated16<4>(v));
  v = fmaxf(v, rotated16<2>(v));
  return fmaxf(v, rotated16<1>(v));
}
__device__ __forceinline__ float sum64(float v) {
  v = sum16(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return xhalf_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Sums of a and b over the TPR lanes of a row, in each of them.  For rows of several waves every thread of the block
// calls it; consecutive calls alternate between the two halves of scratch, so one barrier a call is enough.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float2* scratch, int& half) {
  a = TPR == 16 ? sum16(a) : sum64(a);
  b = TPR == 16 ? sum16(b) : sum64(b);
  if (TPR > kWave) {
    constexpr int kWaves = TPR / kWave;
    float2* s = scratch + half * kWaves;
    half ^= 1;
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      a += s[i].x;
      b += s[i].y;
    }
  }
}

// ---------------------------------------------------------------- 8-bit blocks
// A block's scale is 2^e with the smallest e that brings its largest finite magnitude within the type's range (448 =
// 1.75 2^8, 57344 = 1.75 2^15), kept as the byte e + 127; an all-zero block has e = 0.  e stays at or above -127.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ int block_exponent(float amax, int fp8) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - (fp8 == kFp8E4m3 ? 8 : 15) + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return u == 0 ? 0 : max(e, -127);
}
__device__ __forceinline__ float power2(int e) {  // -127 <= e <= 127
  return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 0x00400000u);
}
// Four values times 2^-e in 8 bits, to nearest even.  Non-finite values become NaN (e5m2 keeps infinities).
__device__ __forceinline__ uint32_t cvt_fp8x4(float a, float b, float c, float d, int fp8) {
  int w = 0;
  if (fp8 == kFp8E4m3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return (uint32_t)w;
}
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], int e, int fp8) {
  const float s = power2(-e);
  return make_uint2(cvt_fp8x4(f[0] * s, f[1] * s, f[2] * s, f[3] * s, fp8),
                    cvt_fp8x4(f[4] * s, f[5] * s, f[6] * s, f[7] * s, fp8));
}

}  // namespace svoo
