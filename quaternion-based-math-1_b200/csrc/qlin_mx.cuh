// 4-bit quaternion weights (OCP microscaling, MXFP4): layout, quantisation and
// dequantisation.
//
// Element format e2m1 (sign, 2 exponent bits, 1 mantissa bit): +-{0, 0.5, 1,
// 1.5, 2, 3, 4, 6}.  32 consecutive input quaternions of one component row
// W_p[o, :] share one E8M0 scale 2^(E - 127):
//
//     E - 127 = floor(log2(max |w|)) - 2,   code = e2m1(w / 2^(E - 127))
//
// rounded to nearest, ties to the even code, saturating at 6 (the quotient is
// below 8).  The power-of-two quotient is exact, so the codes are those of the
// real-number definition.  E is clamped to [0, 254] (a block of zeros has
// E = 0); a block that holds an infinity or a NaN gets zero codes and stands
// for NaNs.
//
// Buffer: a header of kMxHeader bytes (word 0: the largest F of the layer's finite
// blocks; word 1: 255 less the smallest F of those that are not zero), then one record
// per 16 output quaternions (tile) and 32 input quaternions (block), tile-major, blocks
// of one tile contiguous:
//
//     record (1088 bytes) = codes [16 rows][4 octets t][4 components p] words,
//                           then F [16 rows][4 components p] bytes
//
// F = E + 1, or 255 for NaNs, so that the fp32 number with exponent field F is
// normal (twice the scale) or infinite.  Rows and input quaternions past the
// layer's are zero codes with F = 1.
//
// Word (row, t, p) holds the codes of input quaternions 32 b + 8 t + j (j =
// 0..7) of component p, quaternions k and k + 4 (a pair) in its low and high
// half.  The four bits of a code lie where shifts by 0, 3 and 6 and one mask
// bring three of the four pairs to sign and magnitude bits of two bf16 values
// (bit of a half: 8 7 6 magnitude, 15 sign):
//
//     pair 0: 8 7 6, 15    pair 1: 5 4 3, 12    pair 2: 2 1 0, 9
//     pair 3: the rest: 11 10 13, 14
//
// One 16-byte piece holds all four components of eight input quaternions of a
// row, and the pieces that the 32 lanes of an m16 tensor-core operand need are
// two runs of 512 bytes.
#pragma once

#include <type_traits>

#include "qlin_common.cuh"

namespace qlin {

constexpr int kMxBlock = 32;           // input quaternions that share a scale
constexpr int kMxRows = 16;            // output quaternions of a record
constexpr int kMxCodeBytes = kMxRows * kMxBlock * 4 / 2;
constexpr int kMxRecord = kMxCodeBytes + kMxRows * 4;
constexpr int kMxHeader = 128;

// The scale 2^(F - 128) as fp32 (F = 1: the subnormal 2^-127).
__device__ __forceinline__ float mx_scale(uint32_t f) {
  return __uint_as_float(f == 255u ? 0x7FC00000u : (f == 1u ? 0x00400000u : (f - 1u) << 23));
}

// Eight quotients (below 8 in magnitude) as a code word: conversions to e2m1 (to
// nearest, ties to the even code, saturating at 6) pack nibble j = element j,
// whose bits then move to their places, both halves at once.
__device__ __forceinline__ uint32_t mx_pack(const float (&q)[8]) {
  uint32_t n;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(n)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  auto at = [&](int left, uint32_t mask) { return (left >= 0 ? n << left : n >> -left) & (mask | mask << 16); };
  return at(6, 0x01C0u) | at(12, 0x8000u) |                   // pair 0
         at(-1, 0x0038u) | at(5, 0x1000u) |                   // pair 1
         at(-8, 0x0007u) | at(-2, 0x0200u) |                  // pair 2
         at(-3, 0x0C00u) | at(1, 0x2000u) | at(-1, 0x4000u);  // pair 3
}

// Powers of two that the compiler cannot see: left shifts written as products
// with them go to the multiply-add pipe, beside the masks on the integer pipe
// (which alone would bound the expansion).
struct MxPowers {
  uint32_t p1, p3, p6;
  __device__ __forceinline__ MxPowers() {
    asm volatile("mov.u32 %0, 2;" : "=r"(p1));
    asm volatile("mov.u32 %0, 8;" : "=r"(p3));
    asm volatile("mov.u32 %0, 64;" : "=r"(p6));
  }
};

// Eight codes of a word as pairs (k, k + 4) of 16-bit floats: bf16 with the
// code's value times 2^-126, or f16 with its value times 2^-14 (both exact;
// the codes of +-0.5 are subnormal there).
template <bool HALF>
__device__ __forceinline__ void mx_expand(const MxPowers& c, uint32_t w, uint32_t (&r)[4]) {
  const uint32_t w1 = w * c.p1, w3 = w * c.p3, w6 = w * c.p6;
  if constexpr (HALF) {
    constexpr uint32_t kS = 0x80008000u, kM = 0x0E000E00u;
    r[0] = (w & kS) | (w3 & kM);
    r[1] = (w3 & kS) | (w6 & kM);
    r[2] = (w6 & kS) | ((w6 * c.p3) & kM);
    r[3] = (w1 & kS) | ((w >> 4) & 0x02000200u) | (w & 0x0C000C00u);
  } else {
    constexpr uint32_t kSM = 0x81C081C0u;
    r[0] = w & kSM;
    r[1] = w3 & kSM;
    r[2] = w6 & kSM;
    r[3] = (w1 & 0x80008000u) | ((w >> 7) & 0x00400040u) | ((w >> 3) & 0x01800180u);
  }
}

// The values of a word's codes, in order.
__device__ __forceinline__ void mx_values(uint32_t w, float (&v)[8]) {
  uint32_t r[4];
  mx_expand<true>(MxPowers(), w, r);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __half2 h = *reinterpret_cast<const __half2*>(&r[k]);
    v[k] = __low2float(h) * 16384.f;
    v[k + 4] = __high2float(h) * 16384.f;
  }
}

// E of a block whose largest magnitude is amax (finite).
__device__ __forceinline__ uint32_t mx_exponent(float amax) {
  const uint32_t field = __float_as_uint(amax) >> 23;  // floor(log2) + 127; 0 for subnormals
  return field <= 2u ? 0u : field - 2u;
}

// Eight consecutive elements of a row from `at` as they are, zero from `left` on
// (vec: the row pieces are 16-byte aligned).
template <typename T>
struct MxRaw8 {
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* at, int left, bool vec) {
    if (vec && left >= 8) {
#pragma unroll
      for (int u = 0; u < (int)sizeof(T) / 2; ++u) q[u] = ld_cg_v4(reinterpret_cast<const uint4*>(at) + u);
      return;
    }
    T* e = reinterpret_cast<T*>(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j < left ? at[j] : from_f32<T>(0.f);
  }
  __device__ __forceinline__ float get(int j) const { return to_f32(reinterpret_cast<const T*>(q)[j]); }
};

template <typename T>
struct MxPlanes {
  T* w[4];
};

// Quantisation: a warp takes four rows of two neighbouring records, a row of all
// four components per step: 128 bytes in a row of each from eight lanes.  A lane
// holds eight elements of one block, the four lanes of a block share its maximum.
// One pass, the next rows' loads in flight while a warp works on these, everything else
// in registers.  Three CTAs per SM: with all rows at once the tail of the grid reads
// alone.  4096 -> 11008 in bf16 (22.6 MB in, 6 MB out): 11.5 us, 2.5 TB/s, with caches
// cold; about 6.5 us of that are the first loads and the end, and then the integer
// pipe (60 % over the whole launch: conversion, maxima, code words) before HBM.
constexpr int kMxUnitRows = 4;

template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_quantize_kernel(const MxPlanes<const T> src, int64_t ld, int K_g, int N_g, uint8_t* mx, bool vec) {
  const int lane = threadIdx.x & 31;
  const int t = lane & 3, second = (lane >> 2) & 1, p = lane >> 3;
  const int kb = (K_g + kMxBlock - 1) / kMxBlock, row_units = (N_g + kMxRows - 1) / kMxRows * (kMxRows / kMxUnitRows);
  const int b = 2 * ((int)blockIdx.x * 8 + (int)(threadIdx.x >> 5)) + second;  // this lane's block
  uint32_t top = 0, low = 0;
  const int i = b * kMxBlock + 8 * t, left = K_g - i;
  const T* plane = src.w[p] + i;
  MxRaw8<T> raw[kMxUnitRows], next[kMxUnitRows];
  auto fetch = [&](MxRaw8<T>(&to)[kMxUnitRows], int unit) {
#pragma unroll
    for (int u = 0; u < kMxUnitRows; ++u) {
      const int o = unit * kMxUnitRows + u;
      to[u].load(plane + (int64_t)o * ld, o < N_g ? left : 0, vec);
    }
  };
  if ((int)blockIdx.y < row_units) fetch(raw, blockIdx.y);
  for (int unit = blockIdx.y; unit < row_units; unit += gridDim.y) {
    if (unit + (int)gridDim.y < row_units) fetch(next, unit + gridDim.y);
    const int tile = unit / (kMxRows / kMxUnitRows), row0 = unit % (kMxRows / kMxUnitRows) * kMxUnitRows;
    uint8_t* out = mx + kMxHeader + ((int64_t)tile * kb + b) * kMxRecord;
#pragma unroll
    for (int u = 0; u < kMxUnitRows; ++u) {
      const int row = row0 + u;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = raw[u].get(j);
      // magnitudes as integers: the order of finite values, infinities and NaNs above them
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const bool bad = m >= 0x7F800000u;
      const uint32_t e = mx_exponent(__uint_as_float(m));
      const float inv = __uint_as_float((254u - e) << 23);  // 2^(127 - E): E is at most 252
      float q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = bad ? 0.f : v[j] * inv;
      if (!bad) top = max(top, e + 1u);
      if (!bad && m > 0u) low = max(low, 254u - e);
      if (b < kb) {
        *reinterpret_cast<uint32_t*>(out + row * 64 + t * 16 + p * 4) = mx_pack(q);
        if (t == 0) out[kMxCodeBytes + row * 4 + p] = (uint8_t)(bad ? 255u : e + 1u);
      }
      raw[u] = next[u];
    }
  }
  __shared__ uint32_t tops[8], lows[8];
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_max_sync(0xffffffffu, low);
  if (lane == 0) {
    tops[threadIdx.x >> 5] = top;
    lows[threadIdx.x >> 5] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      top = max(top, tops[w]);
      low = max(low, lows[w]);
    }
    // maxima: the same in any order
    atomicMax(reinterpret_cast<unsigned*>(mx), top);
    atomicMax(reinterpret_cast<unsigned*>(mx) + 1, low);
  }
}

// Dequantisation to the four component rows, mapped like the quantisation.
// One rounding (none for fp32, or for bf16 in its normal range).  4096 -> 11008 to bf16
// (6 MB in, 22.6 MB out): 9.3 us, 3.1 TB/s, with caches cold; issue slots (70 %) bound.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_dequantize_kernel(const uint8_t* mx, const MxPlanes<T> dst, int64_t ld, int K_g, int N_g,
                          bool vec) {
  const int lane = threadIdx.x & 31;
  const int t = lane & 3, second = (lane >> 2) & 1, p = lane >> 3;
  const int kb = (K_g + kMxBlock - 1) / kMxBlock, row_units = (N_g + kMxRows - 1) / kMxRows * (kMxRows / kMxUnitRows);
  const int b = 2 * ((int)blockIdx.x * 8 + (int)(threadIdx.x >> 5)) + second;  // this lane's block
  const int i = b * kMxBlock + 8 * t, left = K_g - i;
  if (left <= 0) return;  // (past the last block, too)
  for (int unit = blockIdx.y; unit < row_units; unit += gridDim.y) {
    const int tile = unit / (kMxRows / kMxUnitRows), row0 = unit % (kMxRows / kMxUnitRows) * kMxUnitRows;
    const uint8_t* in = mx + kMxHeader + ((int64_t)tile * kb + b) * kMxRecord;
    uint32_t word[kMxUnitRows], f[kMxUnitRows];
#pragma unroll
    for (int step = 0; step < kMxUnitRows; ++step) {
      const int row = row0 + step;
      word[step] = __ldcg(reinterpret_cast<const uint32_t*>(in + row * 64 + t * 16 + p * 4));
      f[step] = __ldcg(in + kMxCodeBytes + row * 4 + p);
    }
#pragma unroll
    for (int step = 0; step < kMxUnitRows; ++step) {
      const int o = tile * kMxRows + row0 + step;
      if (o >= N_g) continue;
      const float s = mx_scale(f[step]);
      T* at = dst.w[p] + (int64_t)o * ld + i;
      float c[8];
      mx_values(word[step], c);
      __align__(16) T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = from_f32<T>(c[j] * s);
      if (vec && left >= 8) {
#pragma unroll
        for (int u = 0; u < (int)sizeof(T) / 2; ++u)
          reinterpret_cast<uint4*>(at)[u] = reinterpret_cast<const uint4*>(v)[u];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < left) at[j] = v[j];
      }
    }
  }
}

}  // namespace qlin
