// The layer with 4-bit weights for few tokens (decode, small batches; fp32 at
// any size): a stream of the codes through shared memory into warp-level
// tensor-core products (mma m16n8k16, fp32 accumulators).  These, not tcgen05: with
// one to 32 columns of x a 128-row accumulator tile per SM would leave the codes'
// expansion, not the product, as the work, and its hand-over through tensor memory
// costs more than the products (32 tokens, 5120 -> 27648: 39 against 47 us).
//
//     y_a[o] = sum_i sum_p s(a, p) W_p[o, i] x_{a^p}[i]
//
// The weights are the A operand in their stored form: 16 output quaternions x
// 16 input quaternions of one component W_p, expanded from codes in registers
// (no 4x real matrix), so a code is expanded once for all four output
// components and all tokens.  A lane's 16-byte piece of a record holds eight
// input quaternions of a row for all p: the k slots of the operand are
// numbered so that lane t of a group owns input quaternions 8t .. 8t+7 of the
// block in both operands, in the pairs (k, k + 4) that two shifts and masks
// take out of a code word.
//
//   one or two tokens: the eight columns of B are (a, token), column (a, m)
//     holding s(a, p) x_{a^p}[m]: four products of K = 32 give everything.
//   more: the columns are eight tokens of a component plane x_q, sixteen
//     products (a, p) per eight tokens with the sign on A.
//
// Codes expand exactly to bf16 values times 2^-126 (f16: 2^-14), see mx_expand.
//   one or two tokens: those are the operand.  x (bf16) is multiplied by 2^k
//     beforehand, k = 126 minus the exponent of the token's largest value, so
//     that neither overflows nor underflows (a scaling up is exact); the
//     product of a block and component starts from zero and joins the fp32 sum
//     with its scale in one multiply-add per value.
//   more: a packed multiplication by 2^(126 or 14) * scale * 2^-c makes the weights (see
//     MxScaling), and the sums are multiplied by 2^c at the end.
//
// fp32 inputs are split into three bf16 parts of 8 bits each (x = x1 + x2 + x3
// exactly, down to bf16's smallest number); their products go to the same
// accumulator, which starts from zero for every block of 32 input quaternions
// and is added to the fp32 sum outside the tensor core, whose own additions
// truncate.
//
// Bound by the integer pipe and start-up for one token of a wide layer, by latency
// for narrow ones (4096 -> 4096, one token: 4.2 us in a graph, 0.42 of which are bytes),
// by the expansion and the warp-level tensor pipe (50 %) from about 8 tokens on (4096
// -> 4096 at 16 tokens 9.3 us; 5120 -> 27648 at 8 and 16 tokens 17 and 25 us).
#pragma once

#include <type_traits>

#include "qlin_common.cuh"
#include "qlin_mx.cuh"

namespace qlin {

constexpr int kMxWarps = 8;                       // consumer warps of a CTA
constexpr int kMxThreads = 32 * (kMxWarps + 1);   // and the warp that issues the copies
constexpr int kMxRedRow = 65;                     // floats of a reduction row: 64 outputs, padded
constexpr int kMxSmemRank = 256;                  // adapters of up to this rank keep t in shared memory
constexpr int kMxFewBar = 1;                      // named barrier of the consumer warps

__host__ __device__ constexpr int mx_t_rank(int rank) { return rank <= kMxSmemRank ? rank : 0; }

// Sign of component a's product with W_p: bit p of the mask set where it is negative.
__device__ __forceinline__ uint32_t mx_negative(int a) {
  return a == 0 ? 0xEu : (a == 1 ? 0x8u : (a == 2 ? 0x2u : 0x4u));
}

template <typename T>
struct MxOperand {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr int kParts = std::is_same<T, float>::value ? 3 : 1;
};

// An adapter in the CTA-pair kernel (see there): terms of the product per rank, and
// ranks whose terms a stage of 128 holds.
template <typename T>
constexpr int kMxPairParts = MxOperand<T>::kHalf ? 5 : 3;
template <typename T>
constexpr int kMxPairRanks = 128 / kMxPairParts<T> / 8 * 8;

// How a layer's weights become 16-bit operands, times 2^-c.
//   bf16: c = max(0, F0 - 129), with F0 the layer's largest F (c = 0 unless weights reach
//     16); exact.
//   f16: c = F0 - 129, which makes the largest weights 12; exact where no block's scale
//     is below 2^-24 of the largest.  In other layers (`far`) c = F0 - 141, the largest
//     become 49152, by a second multiplication (f16 has no power above 2^15), and scales
//     down to 2^-36 of the largest are exact: all those of fp16 weights below 8192;
//     smaller ones are rounded at 2^-37 of the largest scale.  (Without the distinction, in
//     the CTA-pair kernel: 4096 -> 11008 at 2048 tokens 118 -> 123 us.)
// An adapter's products join the accumulator with B 2^-c: a bound on fp16's c keeps them
// in fp32's range (weights so small, 2^-40 of fp16's steps, are lost in the rounding of y
// anyway).
template <bool HALF>
struct MxScaling {
  int c;
  int off;   // the multiplier of F has the exponent field F - off
  bool far;  // (f16)
  __device__ __forceinline__ MxScaling(const uint8_t* mx, int rank) {
    uint32_t f0, low;
    asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(f0), "=r"(low) : "l"(mx) : "memory");
    if constexpr (HALF) {
      far = (int)f0 - (255 - (int)low) > 24;
      c = max((int)f0 - (far ? 141 : 129), rank > 0 ? -40 : -140);
      off = c + (far ? 111 : 99);  // F - 128 - c + 14 + 15, less the 12 of kMxHalfStep
    } else {
      far = false;
      c = max(0, (int)f0 - 129);
      off = c - 125;  // F - 128 - c + 126 + 127
    }
  }
};

// The packed multiplier of codes with scale F; a NaN block's F saturates at infinity,
// which makes NaNs of its zero codes.
template <bool HALF>
__device__ __forceinline__ uint32_t mx_multiplier(uint32_t f, int off) {
  if constexpr (HALF) {
    const int e = min((int)f - off, 31);
    return (e > 0 ? (uint32_t)e << 10 : (e >= -9 ? 1u << (e + 9) : 0u)) * 0x00010001u;
  } else {
    return (uint32_t)min((int)f - off, 255) * 0x00800080u;
  }
}

template <bool HALF>
__device__ __forceinline__ uint32_t mx_mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (HALF) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

constexpr uint32_t kMxHalfStep = (15u + 12u) * 0x04000400u;  // 2^12, packed f16

// FAR: f16's two multiplications.
template <bool HALF, bool FAR>
__device__ __forceinline__ void mx_expand_scaled(const MxPowers& c, uint32_t w, uint32_t mult, uint32_t (&r)[4],
                                                 uint32_t step = kMxHalfStep) {
  mx_expand<HALF>(c, w, r);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (FAR) r[k] = mx_mul2<true>(r[k], step);
    r[k] = mx_mul2<HALF>(r[k], mult);
  }
}

// d += A B
template <bool HALF>
__device__ __forceinline__ void mx_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d = A B
template <bool HALF>
__device__ __forceinline__ void mx_mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {z,z,z,z};\n\t}"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {z,z,z,z};\n\t}"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// A lane's share of a record: the A operands (weights) of the block's two k16
// steps for all four components.
// (f16: a first multiplication by `step`, 2^12 or 1; 16 tokens, 4096 -> 4096 with rank
// 32: 13.0 us without it, 13.2 with it, 13.5 with a branch on `far`)
template <bool HALF>
__device__ __forceinline__ void mx_load_a(const MxPowers& pw, uint32_t rec, int g, int t, int off, uint32_t step,
                                          uint32_t (&lo)[4][4], uint32_t (&hi)[4][4]) {
  const uint4 wl = lds128(rec + g * 64 + t * 16), wh = lds128(rec + (g + 8) * 64 + t * 16);
  const uint32_t sl = lds32(rec + kMxCodeBytes + g * 4), sh = lds32(rec + kMxCodeBytes + (g + 8) * 4);
  const uint32_t l[4] = {wl.x, wl.y, wl.z, wl.w}, h[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    mx_expand_scaled<HALF, HALF>(pw, l[p], mx_multiplier<HALF>((sl >> (8 * p)) & 255u, off), lo[p], step);
    mx_expand_scaled<HALF, HALF>(pw, h[p], mx_multiplier<HALF>((sh >> (8 * p)) & 255u, off), hi[p], step);
  }
}

// The three bf16 parts of an fp32 value by truncation; a value that is not
// finite is its own first part.
__device__ __forceinline__ void mx_parts(float v, uint32_t (&p)[3]) {
  const uint32_t u = __float_as_uint(v);
  p[1] = p[2] = 0u;
  if ((u & 0x7F800000u) == 0x7F800000u) {
    p[0] = (u >> 16) | ((u & 0x007FFFFFu) ? 0x40u : 0u);
    return;
  }
  p[0] = u >> 16;
  const float r = v - __uint_as_float(u & 0xFFFF0000u);
  const uint32_t ur = __float_as_uint(r);
  p[1] = ur >> 16;
  p[2] = __float_as_uint(r - __uint_as_float(ur & 0xFFFF0000u)) >> 16;
}

// Four consecutive elements.
template <typename T>
__device__ __forceinline__ float4 mx_load4(const T* at, bool vec) {
  if (!vec) return make_float4(to_f32(at[0]), to_f32(at[1]), to_f32(at[2]), to_f32(at[3]));
  if constexpr (sizeof(T) == 4) {
    return ld_cg_f4(at);
  } else {
    uint2 q;
    asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(q.x), "=r"(q.y) : "l"(at) : "memory");
    const T* e = reinterpret_cast<const T*>(&q);
    return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
  }
}

// Input quaternions i and i + 4 of a row in shared memory as B words: out[part][q]
// holds their components q; zero past the layer's.
template <typename T>
__device__ __forceinline__ void mx_arrange_pair(const T* row, int i, int K_g,
                                                uint32_t (&out)[MxOperand<T>::kParts][4]) {
  if constexpr (sizeof(T) == 2) {
    const uint2* at = reinterpret_cast<const uint2*>(row);
    const uint2 a = i < K_g ? at[i] : make_uint2(0u, 0u), b = i + 4 < K_g ? at[i + 4] : make_uint2(0u, 0u);
    out[0][0] = __byte_perm(a.x, b.x, 0x5410);
    out[0][1] = __byte_perm(a.x, b.x, 0x7632);
    out[0][2] = __byte_perm(a.y, b.y, 0x5410);
    out[0][3] = __byte_perm(a.y, b.y, 0x7632);
  } else {
    const float4* at = reinterpret_cast<const float4*>(row);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 a = i < K_g ? at[i] : zero, b = i + 4 < K_g ? at[i + 4] : zero;
    const float va[4] = {a.x, a.y, a.z, a.w}, vb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t pa[3], pb[3];
      mx_parts(va[q], pa);
      mx_parts(vb[q], pb);
#pragma unroll
      for (int s = 0; s < 3; ++s) out[s][q] = pa[s] | pb[s] << 16;
    }
  }
}

// Eight input quaternions 8 oct .. 8 oct + 7 of a row in global memory as B
// words: out[part][q][k] holds component q of quaternions k and k + 4.
template <typename T>
__device__ __forceinline__ void mx_arrange(const T* row, int oct, int K_g, bool vec,
                                           uint32_t (&out)[MxOperand<T>::kParts][4][4]) {
  const int left = K_g - 8 * oct;
  const T* at = row + 32 * (int64_t)oct;
  if constexpr (sizeof(T) == 2) {
    uint32_t w[8][2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j][0] = w[j][1] = 0u;
      if (j < left) {
        if (vec) {
          asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(w[j][0]), "=r"(w[j][1]) : "l"(at + 4 * j) : "memory");
        } else {
          const unsigned short* e = reinterpret_cast<const unsigned short*>(at + 4 * j);
          w[j][0] = e[0] | (uint32_t)e[1] << 16;
          w[j][1] = e[2] | (uint32_t)e[3] << 16;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        out[0][q][k] = __byte_perm(w[k][q >> 1], w[k + 4][q >> 1], (q & 1) ? 0x7632 : 0x5410);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v[2][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = k + 4 * h;
        if (j < left) {
          const float4 f = mx_load4(at + 4 * j, vec);
          v[h][0] = f.x; v[h][1] = f.y; v[h][2] = f.z; v[h][3] = f.w;
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t a[3], b[3];
        mx_parts(v[0][q], a);
        mx_parts(v[1][q], b);
#pragma unroll
        for (int s = 0; s < 3; ++s) out[s][q][k] = a[s] | b[s] << 16;
      }
    }
  }
}

template <typename T>
struct MxFewParams {
  const T* x;
  int64_t ld_x;
  const uint8_t* records;   // [tile][block]
  const uint8_t* mx;        // the codes' header (F0)
  const uint8_t* arranged;  // B words of all tokens (more than two tokens)
  const T* bias;
  const T* lora_b;          // [4 N_g, rank]
  const float* t;           // [M, rank] scaled down projection
  T* y;
  int64_t ld_y;
  int M, K_g, N_g, rank;
  int kb;                   // blocks of a row
  int tiles;                // tiles of 16 output quaternions
  int ring;                 // stages of the ring
  int vec;                  // whole quaternions of x are aligned (one or two tokens: x takes bulk copies)
  int stage_b;              // rows of lora_b come through shared memory
  int vec_b;                // rows of lora_b are whole pieces of 16 or 8 bytes (or 0)
  int after_prologue;       // t comes from the previous kernel, which waited for everything before it
};

// Rows of lora_b in shared memory: padded by 16 bytes, so that neighbouring rows'
// pieces lie in different banks; two buffers for a tile of 64 * WO outputs.
template <typename T>
__host__ __device__ constexpr int mx_b_row(int rank) { return rank * (int)sizeof(T) + 16; }
template <typename T>
__host__ __device__ constexpr int mx_b_bytes(int rank, int wo) { return 2 * 64 * wo * mx_b_row<T>(rank); }
constexpr int kMxMostB = 24 * 1024;  // of the two buffers

// Fetches the rows of lora_b of a tile's outputs n0 .. n0 + 64 WO - 1 (the last one's
// again past the end), by `threads` threads.
template <typename T>
__device__ __forceinline__ void mx_fetch_b(const MxFewParams<T>& prm, uint8_t* dst, int64_t n0, int rows, int thread,
                                           int threads) {
  const int chunks = prm.rank * (int)sizeof(T) / 16;
  for (int k = thread; k < rows * chunks; k += threads) {
    const int row = k / chunks, c = k - row * chunks;
    const int64_t n = min(n0 + row, 4 * (int64_t)prm.N_g - 1);
    cp_async16(smem_u32(dst) + row * mx_b_row<T>(prm.rank) + 16 * c,
               reinterpret_cast<const uint8_t*>(prm.lora_b + n * prm.rank) + 16 * c, 16);
  }
}

// Sums the K split of a tile's outputs (o of 16, a) for a token from the
// reduction rows, adds adapter and bias, and stores.  WARPS rows of partial
// sums per token starting at red (rows of kMxRedRow floats, token-major); `b`: the
// output's row of lora_b in shared memory, or null.
template <int WARPS, typename T>
__device__ __forceinline__ void mx_finish(const MxFewParams<T>& prm, const float* red, int warp_stride, int tok_local,
                                          int col, int64_t m, int64_t n0, float factor, const float* ts,
                                          const uint8_t* b_row) {
  const int64_t n = n0 + col;
  if (m >= prm.M || n >= 4 * (int64_t)prm.N_g) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v += red[w * warp_stride + tok_local * kMxRedRow + col];
  v *= factor;
  if (prm.rank > 0) {
    float l = 0.f;
    const T* b = prm.lora_b + n * prm.rank;
    auto pieces = [&](const auto* row) {
      constexpr int V = (int)(sizeof(*row) / sizeof(T));
      for (int r = 0; r < prm.rank; r += V) {
        const auto q = row[r / V];
        const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int j = 0; j < V; ++j) l = fmaf(ts[r + j], to_f32(e[j]), l);
      }
    };
    if (b_row) pieces(reinterpret_cast<const uint4*>(b_row));
    else if (prm.vec_b == 16) pieces(reinterpret_cast<const uint4*>(b));
    else if (prm.vec_b == 8) pieces(reinterpret_cast<const uint2*>(b));
    else
      for (int r = 0; r < prm.rank; ++r) l = fmaf(ts[r], to_f32(b[r]), l);
    v += l;
  }
  if (prm.bias) v += to_f32(prm.bias[n]);
  prm.y[m * prm.ld_y + n] = from_f32<T>(v);
}

// ---------------------------------------------------------------------------
// one or two tokens
// ---------------------------------------------------------------------------

// G groups of W consumer warps and one copying warp; a group takes a tile at a
// time, its warps every W-th block of it.  The groups share x: with more tiles
// than SMs, three groups keep three tiles of an SM in flight on one staged x
// (5120 -> 27648, one bf16 token: 7.9 us a call, 2.4 TB/s of codes; two CTAs per SM,
// each with its own copy of x, 12.3).  About half of that is start, staging of x and
// the last reduction; in the loop the integer pipe (49 % over the whole launch) and
// issue slots (55 %) bound, not HBM.
//
// Shared memory: a ring per group, x as B words [block][part][sign][q][token][t]
// (both signs, so that no lane flips its operand), x as it came, reduction rows
// (two buffers per group), t, barriers.
template <typename T>
__host__ __device__ constexpr size_t mx_one_raw_bytes(int K_g) { return ((size_t)K_g * 4 * sizeof(T) + 15) / 16 * 16; }
template <typename T>
__host__ __device__ constexpr size_t mx_one_x_bytes(int kb) { return (size_t)kb * MxOperand<T>::kParts * 1024; }

template <typename T, int W, int G>
constexpr size_t mx_one_smem(int M, int K_g, int ring, int rank, int b_bytes) {
  return (size_t)G * ring * (W * kMxRecord + 16) + mx_one_x_bytes<T>((K_g + kMxBlock - 1) / kMxBlock) +
         M * mx_one_raw_bytes<T>(K_g) + G * (2 * W * 2 * kMxRedRow * 4 + b_bytes) + 2 * mx_t_rank(rank) * 4 + 64;
}

// Position in a ring of `stages` stages.
struct MxRing {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++at == stages) {
      at = 0;
      phase ^= 1u;
    }
  }
};

template <typename T, int W, int G>
__global__ void __launch_bounds__(32 * (W + 1) * G)
qlin_mx_one_kernel(const MxFewParams<T> prm) {
  constexpr bool HALF = MxOperand<T>::kHalf;
  constexpr int P = MxOperand<T>::kParts;
  constexpr int kStage = W * kMxRecord;  // a record per warp
  constexpr int kWorkers = 32 * W * G;   // threads that stage x
  constexpr int kAllBar = G + 1;         // named barrier of all consumer warps; group g has 1 + g
  using E = typename std::conditional<sizeof(T) == 2, unsigned short, uint32_t>::type;
  extern __shared__ __align__(128) uint8_t mx_smem[];
  const int S = prm.ring, kb = prm.kb;
  uint8_t* xs = mx_smem + G * S * kStage;
  uint8_t* raw = xs + mx_one_x_bytes<T>(kb);
  const size_t raw_row = mx_one_raw_bytes<T>(prm.K_g);
  const int b_bytes = prm.stage_b ? mx_b_bytes<T>(prm.rank, 1) : 0;
  uint8_t* bs_all = raw + prm.M * raw_row;
  float* red_all = reinterpret_cast<float*>(bs_all + G * b_bytes);
  float* ts = red_all + G * 2 * W * 2 * kMxRedRow;
  uint64_t* bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(ts + 2 * mx_t_rank(prm.rank)) + 7) & ~uintptr_t(7));
  uint64_t* x_full = bars + 2 * G * S;
  uint32_t* largest = reinterpret_cast<uint32_t*>(x_full + 1);  // [2], of the tokens, as bits

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool copies = warp >= W * G;
  const int grp = copies ? warp - W * G : warp / W;
  uint8_t* ring = mx_smem + grp * S * kStage;
  uint64_t* full = bars + 2 * grp * S;
  uint64_t* empty = full + S;
  const int nst = (kb + W - 1) / W;
  // tile = id, id + stride, ...; a CTA's groups are far apart, so that few tiles spread over the SMs
  const int id = (int)blockIdx.x + grp * (int)gridDim.x, stride = G * (int)gridDim.x;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < G * S; ++s) {
      mbar_init(&bars[2 * (s / S) * S + s % S], 1);
      mbar_init(&bars[(2 * (s / S) + 1) * S + s % S], W);
    }
    mbar_init(x_full, 1);
    largest[0] = largest[1] = 0u;
    fence_mbar_init();
  }
  if (!prm.after_prologue) pdl_wait_prior();
  __syncthreads();

  if (copies) {
    if (lane == 0) {
      if (grp == 0 && prm.vec) {  // ahead of the codes: behind them x would be the last to arrive
        const uint32_t row = (uint32_t)prm.K_g * 4 * sizeof(T);
        mbar_arrive_expect_tx(x_full, prm.M * row);
        for (int m = 0; m < prm.M; ++m) bulk_load(raw + m * raw_row, prm.x + m * prm.ld_x, row, x_full);
      }
      MxRing r;
      int issued = 0;
      bool ok = true;
      for (int tile = id; tile < prm.tiles && ok; tile += stride) {
        const uint8_t* src = prm.records + (int64_t)tile * kb * kMxRecord;
        for (int st = 0; st < nst; ++st) {
          if (issued >= S && !mbar_wait(&empty[r.at], r.phase ^ 1u)) {
            ok = false;
            break;
          }
          const uint32_t bytes = min(W, kb - st * W) * kMxRecord;
          mbar_arrive_expect_tx(&full[r.at], bytes);
          bulk_load(ring + r.at * kStage, src + (int64_t)st * kStage, bytes, &full[r.at]);
          r.next(S);
          ++issued;
        }
      }
      // issued copies have landed before the shared memory goes away
      if (grp == 0 && prm.vec) mbar_wait(x_full, 0);
      for (int k = max(0, issued - S); k < issued; ++k) mbar_wait(&full[k % S], (k / S) & 1);
    }
    return;
  }

  bool ok = true;  // a wait that ran out has recorded its error: on without waiting
  if (prm.vec) {
    ok = mbar_wait(x_full, 0);
  } else {  // rows that no bulk copy takes
    for (int m = 0; m < prm.M; ++m)
      for (int k = threadIdx.x; k < 4 * prm.K_g; k += kWorkers)
        reinterpret_cast<E*>(raw + m * raw_row)[k] = *reinterpret_cast<const volatile E*>(prm.x + m * prm.ld_x + k);
    asm volatile("bar.sync %0, %1;" ::"n"(kAllBar), "n"(kWorkers) : "memory");
  }
  // true = sum * factor: F's exponent field makes twice the scale, the codes
  // carry 2^-14 (f16) or, with x's 2^k, 2^(k - 126)
  const int octets = 4 * kb;
  float factor[2] = {8192.f, 8192.f};
  uint32_t up[2] = {0u, 0u};  // 2^k, packed
  if constexpr (!HALF) {
    // k from the largest finite magnitude of a token
#pragma unroll
    for (int tok = 0; tok < 2; ++tok) {
      if (tok >= prm.M) break;
      uint32_t m = 0;
      for (int k = threadIdx.x; k < prm.K_g; k += kWorkers) {
        if constexpr (sizeof(T) == 2) {
          const uint2 v = reinterpret_cast<const uint2*>(raw + tok * raw_row)[k];
          const uint32_t e[4] = {v.x << 16, v.x & 0xFFFF0000u, v.y << 16, v.y & 0xFFFF0000u};
#pragma unroll
          for (int q = 0; q < 4; ++q) m = max(m, (e[q] & 0x7F800000u) == 0x7F800000u ? 0u : e[q] & 0x7F800000u);
        } else {
          const uint4 v = reinterpret_cast<const uint4*>(raw + tok * raw_row)[k];
          const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) m = max(m, (e[q] & 0x7F800000u) == 0x7F800000u ? 0u : e[q] & 0x7F800000u);
        }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == 0 && m > 0u) atomicMax(&largest[tok], m);
    }
    asm volatile("bar.sync %0, %1;" ::"n"(kAllBar), "n"(kWorkers) : "memory");
#pragma unroll
    for (int tok = 0; tok < 2; ++tok) {
      const int k = min(127, 253 - (int)(largest[tok] >> 23));
      factor[tok] = scalbnf(1.f, 125 - k);
      up[tok] = (uint32_t)(127 + k) * 0x00800080u;
    }
  }
  // a thread takes a pair of input quaternions (k, k + 4 of an octet) of a token
  // (with one token the second's columns hold whatever the memory held: no
  // other column sees them)
  for (int idx = threadIdx.x; idx < prm.M * octets * 4; idx += kWorkers) {
    const int tok = idx >= octets * 4 ? 1 : 0, pair = idx - tok * octets * 4, oct = pair >> 2, k = pair & 3;
    uint32_t w[P][4];
    mx_arrange_pair<T>(reinterpret_cast<const T*>(raw + tok * raw_row), 8 * oct + k, prm.K_g, w);
    uint32_t* at = reinterpret_cast<uint32_t*>(xs + ((oct >> 2) * P * 16 + tok) * 64 + (oct & 3) * 16) + k;
#pragma unroll
    for (int s = 0; s < P; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t v = w[s][q];
        if constexpr (!HALF) v = mx_mul2<false>(v, tok ? up[1] : up[0]);
        at[(s * 16 + q * 2) * 16] = v;
        at[(s * 16 + 8 + q * 2) * 16] = v ^ 0x80008000u;
      }
  }
  asm volatile("bar.sync %0, %1;" ::"n"(kAllBar), "n"(kWorkers) : "memory");
  const int g = lane >> 2, t = lane & 3;
  const int a_of = g >> 1, tok_of = g & 1;  // this lane's B column
  uint32_t from[4];
#pragma unroll
  for (int p = 0; p < 4; ++p)
    from[p] = smem_u32(xs) + ((mx_negative(a_of) >> p & 1) * 8 + (a_of ^ p) * 2 + tok_of) * 64 + t * 16;

  float* red = red_all + grp * 2 * W * 2 * kMxRedRow;
  const int gwarp = warp - grp * W, gthread = (int)threadIdx.x - grp * W * 32;
  const MxPowers pw;
  uint32_t byte_up[3];  // F byte p to the exponent field
  asm volatile("mov.u32 %0, 0x00800000;" : "=r"(byte_up[0]));
  asm volatile("mov.u32 %0, 0x00008000;" : "=r"(byte_up[1]));
  asm volatile("mov.u32 %0, 0x00000080;" : "=r"(byte_up[2]));
  MxRing r;
  int buffer = 0;
  for (int tile = id; tile < prm.tiles; tile += stride) {
    uint8_t* bs = bs_all + grp * b_bytes + buffer * (b_bytes / 2);
    if (prm.stage_b) mx_fetch_b<T>(prm, bs, (int64_t)tile * 4 * kMxRows, 64, gthread, 32 * W);
    float acc[4] = {};
    for (int b = gwarp; b < nst * W; b += W) {
      if (ok) ok = mbar_wait(&full[r.at], r.phase);
      if (b < kb) {
        const uint32_t rec = smem_u32(ring) + r.at * kStage + gwarp * kMxRecord;
        const uint4 wl = lds128(rec + g * 64 + t * 16), wh = lds128(rec + (g + 8) * 64 + t * 16);
        const uint32_t sl = lds32(rec + kMxCodeBytes + g * 4), sh = lds32(rec + kMxCodeBytes + (g + 8) * 4);
        const uint32_t l[4] = {wl.x, wl.y, wl.z, wl.w}, h[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t lo[4], hi[4];
          mx_expand<HALF>(pw, l[p], lo);
          mx_expand<HALF>(pw, h[p], hi);
          float d[4];
#pragma unroll
          for (int s3 = 0; s3 < P; ++s3) {
            const uint4 w = lds128(from[p] + (b * P + s3) * 1024);
            if (s3 == 0) mx_mma_first<HALF>(d, lo[0], hi[0], lo[1], hi[1], w.x, w.y);
            else mx_mma<HALF>(d, lo[0], hi[0], lo[1], hi[1], w.x, w.y);
            mx_mma<HALF>(d, lo[2], hi[2], lo[3], hi[3], w.z, w.w);
          }
          const uint32_t fl = p < 3 ? sl * byte_up[p] : sl >> 1, fh = p < 3 ? sh * byte_up[p] : sh >> 1;
          const float ml = __uint_as_float(fl & 0x7F800000u), mh = __uint_as_float(fh & 0x7F800000u);
          acc[0] = fmaf(d[0], ml, acc[0]);
          acc[1] = fmaf(d[1], ml, acc[1]);
          acc[2] = fmaf(d[2], mh, acc[2]);
          acc[3] = fmaf(d[3], mh, acc[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[r.at]);
      r.next(S);
    }
    // lane (g, t): rows g and g + 8, columns (a = t, token 0), (a = t, token 1)
    float* rows = red + buffer * W * 2 * kMxRedRow;
    float* mine = rows + gwarp * 2 * kMxRedRow;
#pragma unroll
    for (int k = 0; k < 4; ++k) mine[(k & 1) * kMxRedRow + 4 * (g + 8 * (k >> 1)) + t] = acc[k];
    if (tile == id && prm.rank > 0) {
      if (prm.after_prologue) pdl_wait_prior();
      // (every group writes the same values)
      for (int k = gthread; k < prm.M * mx_t_rank(prm.rank); k += 32 * W) ts[k] = __ldcg(prm.t + k);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(32 * W) : "memory");
    if (gthread < 64 * prm.M) {
      const int tok = gthread >> 6, col = gthread & 63;
      mx_finish<W>(prm, rows, 2 * kMxRedRow, tok, col, tok, (int64_t)tile * 4 * kMxRows,
                   tok ? factor[1] : factor[0], (prm.rank <= kMxSmemRank ? ts : prm.t) + tok * prm.rank,
                   prm.stage_b ? bs + col * mx_b_row<T>(prm.rank) : nullptr);
    }
    buffer ^= 1;
  }
}

// ---------------------------------------------------------------------------
// B words of many tokens, and the down projection of few
// ---------------------------------------------------------------------------
// arranged[token tile of C][block][part][q][token][t]: C * 4 * parts * 64 bytes a block.
template <typename T>
__device__ __forceinline__ void mx_arrange_one(const T* x, int64_t ld_x, int M, int K_g, int kb, int C, bool vec,
                                               uint8_t* out, int64_t idx) {
  constexpr int P = MxOperand<T>::kParts;
  // consecutive threads: consecutive octets of a token
  const int64_t m = idx / (4 * kb);
  const int oct = (int)(idx - m * 4 * kb);
  const int64_t vt = m / C;
  const int tok = (int)(m - vt * C);
  uint32_t w[P][4][4] = {};
  if (m < M) mx_arrange<T>(x + m * ld_x, oct, K_g, vec, w);
  uint8_t* at = out + ((vt * kb + (oct >> 2)) * P * 4 * C + tok) * 64 + (oct & 3) * 16;
#pragma unroll
  for (int s = 0; s < P; ++s)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4*>(at + (int64_t)(s * 4 + q) * C * 64) =
          make_uint4(w[s][q][0], w[s][q][1], w[s][q][2], w[s][q][3]);
}

constexpr int kMxDownTokens = 4;  // tokens of a down-projection CTA
// Threads of a prologue CTA: the down projection's rounds of dependent loads against
// CTAs whose threads have work (rank 32, rows of 4096, 16 tokens: 13.7 us with 512,
// 15.6 with 256; rank 16, rows of 1024: 7.4 and 6.6).
constexpr int kMxPrologueMost = 512;
inline int mx_prologue_threads(int64_t K_g) { return K_g > 512 ? kMxPrologueMost : 256; }

// Ranks of a down-projection CTA: with four, rows of x are read a quarter as often
// (fp32, 1024 layer, rank 32 at 128 tokens, forward and gradients 114 -> 61 us, together
// with whole 16-byte pieces of lora_b's rows); with one, CTAs are many and short, which
// is better until there are enough of the others (bf16, 4096 layer, rank 32 at 64
// tokens, 128 CTAs of four: 20.9 -> 23.2 us).
constexpr int kMxDownRanksMost = 4;

// Blocks [0, arrange_blocks): the B words.  The rest: t[m, r] = scale x A^T,
// RANKS ranks and kMxDownTokens tokens per block.
template <typename T, int RANKS>
__global__ void __launch_bounds__(kMxPrologueMost)
qlin_mx_prologue_kernel(const T* x, int64_t ld_x, int M, int K_g, int kb, int C, int vec,
                        uint8_t* arranged, int arrange_blocks, int64_t octets,
                        const T* lora_a, int vec_a, int rank, float scale, float* t) {
  pdl_wait_prior();
  pdl_launch_dependents();
  if ((int)blockIdx.x < arrange_blocks) {
    const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx < octets) mx_arrange_one<T>(x, ld_x, M, K_g, kb, C, vec, arranged, idx);
    return;
  }
  constexpr int kSums = RANKS * kMxDownTokens;
  __shared__ float part[kMxPrologueMost / 32][kSums];
  const int b = (int)blockIdx.x - arrange_blocks, groups = (rank + RANKS - 1) / RANKS;
  const int r0 = b % groups * RANKS, m0 = b / groups * kMxDownTokens;
  float s[RANKS][kMxDownTokens] = {};
#pragma unroll(RANKS == 1 ? 2 : 1)
  for (int i = threadIdx.x; i < K_g; i += blockDim.x) {
    float4 av[RANKS];
#pragma unroll
    for (int k = 0; k < RANKS; ++k)  // (past the last rank: that one's again)
      av[k] = mx_load4(lora_a + ((int64_t)min(r0 + k, rank - 1) * K_g + i) * 4, vec_a);
#pragma unroll
    for (int u = 0; u < kMxDownTokens; ++u) {
      if (m0 + u >= M) break;
      const float4 xv = mx_load4(x + (int64_t)(m0 + u) * ld_x + 4 * (int64_t)i, vec);
#pragma unroll
      for (int k = 0; k < RANKS; ++k)
        s[k][u] = fmaf(av[k].x, xv.x, fmaf(av[k].y, xv.y, fmaf(av[k].z, xv.z, fmaf(av[k].w, xv.w, s[k][u]))));
    }
  }
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s[k / kMxDownTokens][k % kMxDownTokens] +=
        __shfl_xor_sync(0xffffffffu, s[k / kMxDownTokens][k % kMxDownTokens], d);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < kSums; ++k) part[threadIdx.x >> 5][k] = s[k / kMxDownTokens][k % kMxDownTokens];
  __syncthreads();
  const int r = r0 + (int)threadIdx.x / kMxDownTokens, m = m0 + (int)threadIdx.x % kMxDownTokens;
  if (threadIdx.x < kSums && r < rank && m < M) {
    float v = 0.f;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) v += part[w][threadIdx.x];
    t[(int64_t)m * rank + r] = scale * v;
  }
}

// ---------------------------------------------------------------------------
// more tokens: NT groups of eight per tile, WO tiles of output quaternions per
// CTA (WO warps side by side, kMxWarps / WO along the blocks)
// ---------------------------------------------------------------------------
// Records of the adjoint, conj(W)^T 2^-c, for fp32 gradients: the same 16 x 32
// quaternions as bf16 pairs (k, k + 4) ready for the operand,
// [component][16 rows][4 octets][4 words] (a code's value times its scale is exact
// in bf16).
constexpr int kMxWideRecord = 4 * kMxRows * 4 * 16;

template <bool HALF>
__device__ __forceinline__ void mx_load_a_wide(uint32_t rec, int g, int t, uint32_t (&lo)[4][4], uint32_t (&hi)[4][4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint4 l = lds128(rec + p * 1024 + (g * 4 + t) * 16), h = lds128(rec + p * 1024 + ((g + 8) * 4 + t) * 16);
    lo[p][0] = l.x; lo[p][1] = l.y; lo[p][2] = l.z; lo[p][3] = l.w;
    hi[p][0] = h.x; hi[p][1] = h.y; hi[p][2] = h.z; hi[p][3] = h.w;
  }
}

// WIDE: the records are wide ones.
template <typename T, int NT, int WO, bool WIDE>
struct MxManyCfg {
  static constexpr int kP = MxOperand<T>::kParts;
  static constexpr int kRecord = WIDE ? kMxWideRecord : kMxRecord;
  static constexpr int kC = 8 * NT;                      // tokens of a tile
  static constexpr int kWK = kMxWarps / WO;              // blocks of a stage
  static constexpr int kXBlock = kP * 4 * kC * 64;       // B words of a block
  static constexpr int kStage = kWK * (WO * kRecord + kXBlock);
  static constexpr int kRed = kMxWarps * 8 * kMxRedRow * 4;  // partial sums of eight tokens
  static constexpr int kFixed = 2 * kRed + 64;  // without t and rows of lora_b
  static_assert(kStage % 16 == 0, "copies of whole 16-byte pieces");
};

template <typename T, int NT, int WO, bool WIDE>
constexpr size_t mx_many_smem(int ring, int rank, int b_bytes) {
  using Cfg = MxManyCfg<T, NT, WO, WIDE>;
  return (size_t)ring * (Cfg::kStage + 16) + Cfg::kFixed + (size_t)Cfg::kC * mx_t_rank(rank) * 4 + b_bytes;
}

template <typename T, int NT, int WO, bool WIDE>
__global__ void __launch_bounds__(kMxThreads, NT == 1 && sizeof(T) == 2 ? 2 : 1)
qlin_mx_many_kernel(const MxFewParams<T> prm) {
  using Cfg = MxManyCfg<T, NT, WO, WIDE>;
  constexpr bool HALF = MxOperand<T>::kHalf;
  constexpr int P = Cfg::kP, C = Cfg::kC, WK = Cfg::kWK, kRecord = Cfg::kRecord;
  extern __shared__ __align__(128) uint8_t mx_smem[];
  const int S = prm.ring, kb = prm.kb;
  const int b_bytes = prm.stage_b ? mx_b_bytes<T>(prm.rank, WO) : 0;
  uint8_t* bs_both = mx_smem + S * Cfg::kStage;
  float* red = reinterpret_cast<float*>(bs_both + b_bytes);
  float* ts = red + 2 * kMxWarps * 8 * kMxRedRow;
  uint64_t* full = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(ts + C * mx_t_rank(prm.rank)) + 7) & ~uintptr_t(7));
  uint64_t* empty = full + S;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nst = (kb + WK - 1) / WK;
  const int groups = (prm.tiles + WO - 1) / WO;           // CTA tiles along the outputs
  const int total = groups * ((prm.M + C - 1) / C);
  const int my_tiles = (int)blockIdx.x < total ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kMxWarps);
    }
    fence_mbar_init();
  }
  pdl_wait_prior();  // the B words and t
  __syncthreads();

  if (warp == kMxWarps) {
    if (lane == 0) {
      MxRing r;
      int issued = 0;
      bool ok = true;
      for (int j = 0; j < my_tiles && ok; ++j) {
        const int id = (int)blockIdx.x + j * (int)gridDim.x;
        const int64_t vt = id / groups, tile0 = (int64_t)(id - (int)vt * groups) * WO;
        for (int st = 0; st < nst; ++st) {
          const int s = r.at;
          if (issued >= S && !mbar_wait(&empty[s], r.phase ^ 1u)) {
            ok = false;
            break;
          }
          const int b0 = st * WK, nb = min(WK, kb - b0);
          const int rows = min(WO, prm.tiles - (int)tile0);
          uint8_t* dst = mx_smem + s * Cfg::kStage;
          mbar_arrive_expect_tx(&full[s], nb * (rows * kRecord + Cfg::kXBlock));
          for (int w = 0; w < rows; ++w)
            bulk_load(dst + w * WK * kRecord, prm.records + ((tile0 + w) * kb + b0) * kRecord, nb * kRecord, &full[s]);
          bulk_load(dst + WO * WK * kRecord, prm.arranged + (vt * kb + b0) * Cfg::kXBlock, nb * Cfg::kXBlock,
                    &full[s]);
          r.next(S);
          ++issued;
        }
      }
      for (int k = max(0, issued - S); k < issued; ++k) mbar_wait(&full[k % S], (k / S) & 1);
    }
    return;
  }

  const MxScaling<HALF> sc(prm.mx, 0);
  const float factor = scalbnf(1.f, sc.c);
  const uint32_t step = sc.far ? kMxHalfStep : 0x3C003C00u;
  const int g = lane >> 2, t = lane & 3;
  const int wo = warp / WK, wk = warp - wo * WK;
  const MxPowers pw;
  MxRing r;
  int round = 0;
  bool ok = true;
  for (int j = 0; j < my_tiles; ++j) {
    const int id = (int)blockIdx.x + j * (int)gridDim.x;
    const int64_t vt = id / groups, tile0 = (int64_t)(id - (int)vt * groups) * WO;
    uint8_t* bs = bs_both + (j & 1) * (b_bytes / 2);
    if (prm.stage_b) mx_fetch_b<T>(prm, bs, tile0 * 4 * kMxRows, 64 * WO, threadIdx.x, 32 * kMxWarps);
    if (mx_t_rank(prm.rank) > 0 && (j == 0 || id / groups != (id - (int)gridDim.x) / groups)) {
      // t of this token tile, once every thread is past the tile before; the
      // barrier after the products orders it before its readers
      asm volatile("bar.sync %0, %1;" ::"n"(kMxFewBar), "n"(32 * kMxWarps) : "memory");
      const int64_t first = vt * C * prm.rank;
      const int count = (int)min((int64_t)C, prm.M - vt * C) * prm.rank;
      for (int k = 4 * threadIdx.x; k < count; k += 4 * 32 * kMxWarps)
        cp_async16(smem_u32(ts + k), prm.t + first + k, 4 * min(4, count - k));
    }
    float acc[NT][4][4] = {};
    for (int st = 0; st < nst; ++st) {
      const int s = r.at;
      if (ok) ok = mbar_wait(&full[s], r.phase);
      if (st * WK + wk < kb && tile0 + wo < prm.tiles) {
        const uint32_t base = smem_u32(mx_smem) + s * Cfg::kStage;
        uint32_t lo[4][4], hi[4][4];
        if constexpr (WIDE) mx_load_a_wide<HALF>(base + (wo * WK + wk) * kRecord, g, t, lo, hi);
        else mx_load_a<HALF>(pw, base + (wo * WK + wk) * kRecord, g, t, sc.off, step, lo, hi);
        const uint32_t xb = base + WO * WK * kRecord + wk * Cfg::kXBlock + g * 64 + t * 16;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4][4] = {};
#pragma unroll
          for (int s3 = 0; s3 < P; ++s3)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint4 w = lds128(xb + ((s3 * 4 + q) * C + nt * 8) * 64);
#pragma unroll
              for (int a = 0; a < 4; ++a) {
                const int p = a ^ q;
                const bool neg = (a == 0 && p != 0) || (a == 1 && p == 3) || (a == 2 && p == 1) || (a == 3 && p == 2);
                const uint32_t f = neg ? 0x80008000u : 0u;
                float(&to)[4] = P > 1 ? d[a] : acc[nt][a];
                mx_mma<HALF>(to, lo[p][0] ^ f, hi[p][0] ^ f, lo[p][1] ^ f, hi[p][1] ^ f, w.x, w.y);
                mx_mma<HALF>(to, lo[p][2] ^ f, hi[p][2] ^ f, lo[p][3] ^ f, hi[p][3] ^ f, w.z, w.w);
              }
            }
          if constexpr (P > 1)
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
              for (int k = 0; k < 4; ++k) acc[nt][a][k] += d[a][k];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      r.next(S);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt, ++round) {
      // eight tokens at a time through one of two buffers
      float* buf = red + (round & 1) * kMxWarps * 8 * kMxRedRow;
      float* mine = buf + warp * 8 * kMxRedRow;
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mine[(2 * t + (k & 1)) * kMxRedRow + 4 * (g + 8 * (k >> 1)) + a] = acc[nt][a][k];
      asm volatile("cp.async.wait_all;" ::: "memory");
      asm volatile("bar.sync %0, %1;" ::"n"(kMxFewBar), "n"(32 * kMxWarps) : "memory");
      for (int k = threadIdx.x; k < 8 * 64 * WO; k += 32 * kMxWarps) {
        const int col = k & 63, w = (k >> 6) % WO, tok = (k >> 6) / WO;
        const int64_t m = vt * C + nt * 8 + tok;
        mx_finish<WK>(prm, buf + w * WK * 8 * kMxRedRow, 8 * kMxRedRow, tok, col, m,
                     (tile0 + w) * 4 * kMxRows, factor,
                     (prm.rank <= kMxSmemRank ? ts : prm.t + vt * C * prm.rank) + (nt * 8 + tok) * prm.rank,
                     prm.stage_b ? bs + (64 * w + col) * mx_b_row<T>(prm.rank) : nullptr);
      }
    }
  }
}

}  // namespace qlin
