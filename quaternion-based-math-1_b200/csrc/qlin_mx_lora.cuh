// The adapter's products around a layer with 4-bit weights.
//
//     t  = s x A^T          [M, r]      u  = s gy B           [M, r]
//     dA = u^T x            [r, K]      dB = gy^T t           [N, r]
//     dbias = sum_m gy[m]   [N]
//
// t and u are kept as parts (or in fp32): rounded to one they would add an error of the
// size of the results' own rounding.  The CTA-pair kernel takes them as three bf16 parts
// (exact), dA and dB as three bf16 ones or two f16 ones with a power of two per rank and
// 16 tokens (mx_top_scale).  x and gy are read once for t and u and once for the
// gradients, which bounds the down projections; the products are warp-level tensor-core
// ones (m16n8k16) whose k slots are numbered so that a lane reads eight consecutive
// elements of a row in one 16-byte piece for both operands (2 M r (K + N) operations are
// too few for tcgen05 tiles: rank 32 fills a quarter of one).
//
// 4096 layer, 2048 bf16 tokens, rank 32 (x and gy: 16.8 MB each), each launch by
// itself: t in the forward pass 10.0 us, everything turned 6.8 us, t and u 14.5 us
// (2.3 TB/s), dA, dB and dbias 20.1 us (15.0 with two parts: their products bound it) and
// the sum of their partial sums 5.7 us.  The first runs under the product's start, dA and
// dB partly beside the input gradient's end.
//
// (Inputs are not declared restrict: the compiler may read through such pointers
// before the dependency wait.)
#pragma once

#include "qlin_common.cuh"
#include "qlin_mx_few.cuh"

namespace qlin {

// out[n] = sum_m g[m, n]
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_column_sum_kernel(const T* g, int64_t ld_g, T* out, int64_t M, int64_t N) {
  __shared__ float part[8][32];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + tx;
  float s = 0.f;
  if (n < N)
    for (int64_t m = ty; m < M; m += 8) s += to_f32(g[m * ld_g + n]);
  part[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && n < N) {
#pragma unroll
    for (int u = 1; u < 8; ++u) s += part[u][tx];
    out[n] = from_f32<T>(s);
  }
}

constexpr int kMxTurnRows = 64;  // output quaternions of a step

// What the gradients need turned, in one launch: blocks [0, steps) make the
// components of conj(W)^T 2^-c (16-bit types: rows of ld elements; fp32: the wide
// records of qlin_mx_few.cuh at dst.w[0]), the next a_blocks A^T, the rest B^T
// (rows of ld_bt elements, zero past B's rows).  A step is 64 output x 32 input quaternions; a thread takes two
// neighbouring output quaternions, eight input quaternions and two components,
// so that the turned pairs go to shared memory as words, a warp's in a row.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_turn_all_kernel(const uint8_t* mx, const MxPlanes<T> dst, int64_t ld, int K_g, int N_g,
                        int64_t steps, const T* a, T* at, int64_t a_rows, int64_t a_cols,
                        const T* b, T* bt, int64_t b_rows, int64_t b_cols, int64_t ld_bt,
                        int64_t a_blocks) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  __shared__ __align__(16) uint32_t turned[4 * kMxBlock][36];  // [component, input quaternion][pair of outputs]
  pdl_wait_prior();
  pdl_launch_dependents();
  if ((int64_t)blockIdx.x >= steps) {
    const bool first = (int64_t)blockIdx.x < steps + a_blocks;
    const int64_t k = ((int64_t)blockIdx.x - steps - (first ? 0 : a_blocks)) * 256 + threadIdx.x;
    // consecutive threads write consecutive elements
    if (first) {
      if (k < a_rows * a_cols) at[k] = a[(k % a_rows) * a_cols + k / a_rows];
    } else if (k < ld_bt * b_cols) {
      const int64_t r = k % ld_bt;
      bt[k] = r < b_rows ? b[r * b_cols + k / ld_bt] : from_f32<T>(0.f);
    }
    return;
  }
  const int64_t kb = (K_g + kMxBlock - 1) / kMxBlock, tiles = (N_g + kMxRows - 1) / kMxRows;
  const int64_t og = blockIdx.x / kb, blk = blockIdx.x - og * kb;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = warp & 3, ph = warp >> 2;
  const MxScaling<HALF> sc(mx, a_rows > 0 ? 1 : 0);
  const int row = 2 * lane;  // of 64
  const int64_t tile = 4 * og + row / kMxRows;
  uint2 w[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
  uint32_t f[2] = {0u, 0u};
  if (tile < tiles) {
    const uint8_t* rec = mx + kMxHeader + (tile * kb + blk) * kMxRecord;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = row % kMxRows + u;
      w[u] = *reinterpret_cast<const uint2*>(rec + r * 64 + t * 16 + ph * 8);
      f[u] = *reinterpret_cast<const uint16_t*>(rec + kMxCodeBytes + r * 4 + ph * 2);
    }
  }
  const MxPowers pw;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int p = 2 * ph + h;
    uint32_t e[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t word = h ? w[u].y : w[u].x;
      const uint32_t mult = mx_multiplier<HALF>((f[u] >> (8 * h)) & 255u, sc.off) ^ (p ? 0x80008000u : 0u);
      if (HALF && sc.far) mx_expand_scaled<HALF, HALF>(pw, word, mult, e[u]);
      else mx_expand_scaled<HALF, false>(pw, word, mult, e[u]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      turned[p * kMxBlock + 8 * t + k][lane] = __byte_perm(e[0][k], e[1][k], 0x5410);
      turned[p * kMxBlock + 8 * t + k + 4][lane] = __byte_perm(e[0][k], e[1][k], 0x7632);
    }
  }
  __syncthreads();
  if constexpr (sizeof(T) == 4) {
    // words (k, k + 4) of an octet of outputs, by [input tile][output block]: two
    // tiles of 16 input quaternions, two blocks of 32 output quaternions
    const int64_t in_tiles = (K_g + kMxRows - 1) / kMxRows, out_blocks = (N_g + kMxBlock - 1) / kMxBlock;
    uint8_t* records = reinterpret_cast<uint8_t*>(dst.w[0]);
    for (int k = threadIdx.x; k < 4 * 4 * kMxRows * 16; k += 256) {
      const int word = k & 3, t = (k >> 2) & 3, r = (k >> 4) & 15, p = (k >> 8) & 3, half = (k >> 10) & 1, bl = k >> 11;
      const int64_t it = 2 * blk + half, ob = 2 * og + bl;
      if (it >= in_tiles || ob >= out_blocks) continue;
      const uint32_t* row = turned[p * kMxBlock + kMxRows * half + r];
      const int o = 32 * bl + 8 * t + word;  // and o + 4
      const uint32_t lo = row[o >> 1], hi = row[(o + 4) >> 1];
      *reinterpret_cast<uint32_t*>(records + (it * out_blocks + ob) * kMxWideRecord + ((p * kMxRows + r) * 4 + t) * 16 +
                                   word * 4) = __byte_perm(lo, hi, (o & 1) ? 0x7632 : 0x5410);
    }
  } else {
    // 16-byte pieces: eight output quaternions of a row (rows of ld, a multiple of 8)
#pragma unroll
    for (int k = threadIdx.x; k < 4 * kMxBlock * 8; k += 256) {
      const int piece = k & 7, i = (k >> 3) & 31, p = k >> 8;
      const int64_t o = og * kMxTurnRows + 8 * piece, in = blk * kMxBlock + i;
      if (o < ld && in < K_g)
        *reinterpret_cast<uint4*>(dst.w[p] + in * ld + o) =
            *reinterpret_cast<const uint4*>(&turned[p * kMxBlock + i][4 * piece]);
    }
  }
}

// dst rows of ld_d elements (ld_d >= cols), zero past cols: rows that no 16-byte
// load takes.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_repack_kernel(const T* src, int64_t ld_s, T* dst, int64_t ld_d, int64_t rows,
                      int64_t cols) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (k >= rows * ld_d) return;
  const int64_t r = k / ld_d, c = k - r * ld_d;
  dst[k] = c < cols ? src[r * ld_s + c] : from_f32<T>(0.f);
}

// ---------------------------------------------------------------------------
// 16-bit down projections: t = scale x A^T
// ---------------------------------------------------------------------------
constexpr int kMxDownRows = 16;   // tokens of a CTA
constexpr int kMxDownRanks = 32;  // ranks of a CTA

// Parts of t and u for dA and dB: bf16's three are exact, f16's two hold 22 bits.  (Two
// bf16 parts, 17 bits: results off by 6e-5 of their norm more than fp32 sums leave, the
// 4096 layer's training step at 2048 tokens 153 us in place of 155.)
template <typename T>
constexpr int kMxTurnedParts = std::is_same<T, __half>::value ? 2 : 3;

template <typename T>
struct MxDownJob {
  const T* x;      // [M, ld_x]
  int64_t ld_x;
  const T* a;      // [rank, ld_a]
  int64_t ld_a;    // (both: 16-byte aligned rows of K elements)
  int K;           // a multiple of 8: zero past the product's terms
  float scale;
  __nv_bfloat16* parts;  // [M, kMxPairParts<T> * ld_parts], the CTA-pair kernel's terms: zero past rank; or null
  T* turned;       // [kMxTurnedParts<T>][rows][M_pad]: parts, the largest first, transposed; or null
  uint8_t* tops;   // f16: [M_pad / 16][rows]: exponent fields of the groups of 16 tokens (see mx_top_scale)
  int rank, ld_parts, rows;
  int rank_tiles;  // ceil(max(ld_parts, rows) / 32)
  int blocks;
};

// f16 parts of a rank and 16 tokens are multiplied by the power of two that brings
// their largest finite magnitude, of exponent field `top`, to 2^14 .. 2^15: unscaled,
// both parts would end at 2^-24, and u is far smaller early in a training (B starts at
// zero) or with small gradients.  `top` is at least kMxLeastTop (the factor stays an
// fp32 number); 0: the group has no finite value but zeros.
constexpr int kMxLeastTop = 14;
__device__ __forceinline__ float mx_top_scale(int top) {
  return top ? __uint_as_float((uint32_t)(268 - top) << 23) : 1.f;
}

constexpr int kMxDownStages = 4;
constexpr int kMxDownPieces = 6;  // 16-byte pieces of a lane and stage: two tokens, four ranks
constexpr int kMxDownSmem = kMxDownStages * kMxDownPieces * 256 * 16;

// A CTA: 16 tokens x 32 ranks, its eight warps every eighth piece of 32 terms.
// Tokens and ranks past the last read the last one's row; what comes of them is
// replaced by zeros.  A lane fetches what it will multiply itself, asynchronously
// and up to three pieces ahead, into slots of its own: no barrier in the loop, and
// 24 loads in flight however the compiler spends its registers.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_down_kernel(const __grid_constant__ MxDownJob<T> job0, const __grid_constant__ MxDownJob<T> job1, int M,
                    int M_pad) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t mx_smem[];
  __shared__ float red[8][kMxDownRows][kMxDownRanks + 1];
  pdl_wait_prior();
  pdl_launch_dependents();
  const bool first = (int)blockIdx.x < job0.blocks;
  const MxDownJob<T>& job = first ? job0 : job1;
  const int id = (int)blockIdx.x - (first ? 0 : job0.blocks);
  const int m0 = id / job.rank_tiles * kMxDownRows, r0 = id % job.rank_tiles * kMxDownRanks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float acc[4][4] = {};
  if (r0 < job.rank && m0 < M) {
    const T* xl = job.x + (int64_t)min(m0 + g, M - 1) * job.ld_x;
    const T* xh = job.x + (int64_t)min(m0 + g + 8, M - 1) * job.ld_x;
    const T* ar[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) ar[n] = job.a + (int64_t)min(r0 + 8 * n + g, job.rank - 1) * job.ld_a;
    constexpr int kStep = 32 * 8;
    const uint32_t slots = smem_u32(mx_smem) + threadIdx.x * 16;
    int k = 32 * warp + 8 * t;   // next to fetch
    MxRing in, out;
    auto fetch = [&]() {
      const uint32_t at = slots + in.at * kMxDownPieces * 256 * 16;
      const int bytes = k < job.K ? 16 : 0, from = k < job.K ? k : 0;
      // (the slot's values were consumed by products issued before: their registers are read)
      cp_async16(at, xl + from, bytes);
      cp_async16(at + 256 * 16, xh + from, bytes);
#pragma unroll
      for (int n = 0; n < 4; ++n) cp_async16(at + (2 + n) * 256 * 16, ar[n] + from, bytes);
      asm volatile("cp.async.commit_group;" ::: "memory");
      k += kStep;
      in.next(kMxDownStages);
    };
#pragma unroll
    for (int u = 0; u < kMxDownStages - 1; ++u) fetch();
    for (int done = 32 * warp; done < job.K; done += kStep) {
      fetch();
      asm volatile("cp.async.wait_group %0;" ::"n"(kMxDownStages - 1) : "memory");
      const uint32_t at = slots + out.at * kMxDownPieces * 256 * 16;
      out.next(kMxDownStages);
      const uint4 lo = lds128(at), hi = lds128(at + 256 * 16);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint4 b = lds128(at + (2 + n) * 256 * 16);
        mx_mma<HALF>(acc[n], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
        mx_mma<HALF>(acc[n], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) red[warp][g + 8 * (q >> 1)][8 * n + 2 * t + (q & 1)] = acc[n][q];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    // the parts of (token, rank); ranks fastest for `parts`, tokens fastest for `turned`
#pragma unroll
    for (int way = 0; way < 2; ++way) {
      if (way == 0 ? !job.parts : !job.turned) continue;
      const int k = threadIdx.x + 256 * u;
      const int m = way == 0 ? k >> 5 : k & 15, r = way == 0 ? k & 31 : k >> 4;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += red[w][m][r];
      v = m0 + m < M && r0 + r < job.rank ? v * job.scale : 0.f;
      if (HALF && way == 1) {  // 16 consecutive lanes: the tokens of a rank
        const uint32_t bits = __float_as_uint(v) & 0x7FFFFFFFu;
        uint32_t most = bits < 0x7F800000u ? bits : 0u;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
        const int top = most ? max((int)(most >> 23), kMxLeastTop) : 0;
        if (m == 0 && r0 + r < job.rows) job.tops[(int64_t)(m0 / kMxDownRows) * job.rows + r0 + r] = (uint8_t)top;
        v *= mx_top_scale(top);
      }
      if (way == 0) {
        if (m0 + m < M && r0 + r < job.ld_parts) {
          // (an infinite or NaN first part stands alone)
          const __nv_bfloat16 p0 = __float2bfloat16_rn(v);
          const float rest = isfinite(to_f32(p0)) ? v - to_f32(p0) : 0.f;
          const __nv_bfloat16 p1 = __float2bfloat16_rn(rest), p2 = __float2bfloat16_rn(rest - to_f32(p1));
          // [stage][part][rank of the stage]
          const int first = (r0 + r) / kMxPairRanks<T> * kMxPairRanks<T>, ranks = min(kMxPairRanks<T>, job.ld_parts - first);
          __nv_bfloat16* at = job.parts + ((int64_t)(m0 + m) * job.ld_parts + first) * kMxPairParts<T> + (r0 + r - first);
          at[0] = p0;
          at[ranks] = p1;
          at[2 * ranks] = p2;
          if (HALF) {
            at[3 * ranks] = isfinite(to_f32(p0)) ? p0 : __float2bfloat16_rn(0.f);
            at[4 * ranks] = p1;
          }
        }
      } else if (r0 + r < job.rows) {
        T* at = job.turned + (int64_t)(r0 + r) * M_pad + m0 + m;
#pragma unroll
        for (int part = 0; part < kMxTurnedParts<T>; ++part, at += (int64_t)job.rows * M_pad) {
          const T p = from_f32<T>(v);
          *at = p;
          v -= to_f32(p);
          if (!isfinite(v)) v = 0.f;  // (an infinite or NaN part stands alone)
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit gradients: out = (sum of the parts) X, sums over the tokens
// ---------------------------------------------------------------------------
constexpr int kMxOuterCols = 128;   // columns of X of a CTA, 32 per warp
constexpr int kMxOuterTokens = 32;  // tokens of a step
constexpr int kMxOuterRows = 64;    // rows of the result of a CTA (groups of 16)
constexpr int kMxOuterStages = 4;
constexpr int kMxOuterXBytes = kMxOuterTokens * kMxOuterCols * 2;
constexpr int kMxOuterTops = 2 * kMxOuterRows;  // bytes: f16's exponents of a step's two groups of 16 tokens

// Bytes of a stage: X, the exponents, the parts of up to kMxOuterRows rows.
template <typename T>
__host__ __device__ constexpr int mx_outer_stage(int rows) {
  return kMxOuterXBytes + kMxOuterTops + kMxTurnedParts<T> * (rows < kMxOuterRows ? rows : kMxOuterRows) * kMxOuterTokens * 2;
}

template <typename T>
struct MxOuterJob {
  const T* turned;  // [kMxTurnedParts<T>][rows][M_pad]; fp32: [M][rows]
  const uint8_t* tops;  // f16: of the parts, see MxDownJob
  const T* X;       // [M, ld], 16-byte aligned rows
  int64_t ld;
  int cols, rows;   // rows: a multiple of 16
  int col_tiles, row_tiles, splits;
  int blocks;
  float* partial;   // [splits][rows][cols]
  float* sums;      // [splits][cols] column sums of X, or null
};

// The packed f16 factor 2^(top - row_top) (0 below f16's numbers) that brings a group's
// parts to their row's power of two.
__device__ __forceinline__ uint32_t mx_top_factor(int top, int row_top) {
  const int e = top ? 15 + top - row_top : 1;  // (a group of zeros, infinities and NaNs: any factor)
  return (e > 0 ? (uint32_t)e << 10 : (e > -10 ? 1u << (9 + e) : 0u)) * 0x00010001u;
}

// Four warps: 32 columns each, all rows.  X and the rows of all parts come through
// a ring of shared memory steps (32 tokens x 128 columns; 16-byte chunks permuted
// within a row of X so that the transposing loads of eight tokens two apart are
// free of conflicts).
//
// f16: a CTA brings the parts of a row to the power of two of the row's largest group
// among its own tokens (one packed multiplication per pair; what falls below f16 is
// 2^-39 of that largest value) and undoes it on the sums.
//
// beside: the launch before is the CTA-pair kernel, which needs nothing from this one
// and lets it start only when the down projections have ended.  CTAs then take the SMs
// that its last wave leaves free; the last CTA waits for its end, so that whatever
// waits for this kernel has waited for that one too.
template <typename T>
__global__ void __launch_bounds__(128)
qlin_mx_outer_kernel(const __grid_constant__ MxOuterJob<T> job0, const __grid_constant__ MxOuterJob<T> job1, int M,
                     int M_pad, int beside) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  constexpr int kParts = kMxTurnedParts<T>;
  extern __shared__ __align__(128) uint8_t mx_smem[];
  if (!beside) pdl_wait_prior();
  pdl_launch_dependents();
  const bool first = (int)blockIdx.x < job0.blocks;
  const MxOuterJob<T>& job = first ? job0 : job1;
  int id = (int)blockIdx.x - (first ? 0 : job0.blocks);
  const int ct = id % job.col_tiles;
  id /= job.col_tiles;
  const int rt = id % job.row_tiles, split = id / job.row_tiles;
  const int steps = M_pad / kMxOuterTokens;
  const int s0 = (int)((int64_t)steps * split / job.splits), s1 = (int)((int64_t)steps * (split + 1) / job.splits);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int c0 = ct * kMxOuterCols, row0 = rt * kMxOuterRows;
  const int rows = min(kMxOuterRows, job.rows - row0), groups = rows / 16;
  // what this thread fetches of a step: a chunk of X of four tokens, and a chunk of
  // up to two rows of every part
  const int tok = threadIdx.x >> 4, chunk = threadIdx.x & 15;  // tokens tok + 8 u
  const int left = min(8, job.cols - (c0 + 8 * chunk));        // elements of the chunk inside
  const int bytes = left > 0 ? 2 * left : 0;
  const T* xp = job.X + (int64_t)(s0 * kMxOuterTokens + tok) * job.ld + (left > 0 ? c0 + 8 * chunk : 0);
  const int64_t x_eight = 8 * job.ld;
  uint32_t x_at[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) x_at[u] = (tok + 8 * u) * 256 + ((chunk ^ ((tok & 1) | u << 1)) << 4);
  const int ar = threadIdx.x >> 2;  // rows ar and ar + 32
  const T* ap = job.turned + (int64_t)(row0 + min(ar, rows - 1)) * M_pad + s0 * kMxOuterTokens + 8 * (threadIdx.x & 3);
  const int64_t part_off = (int64_t)job.rows * M_pad, row32 = 32 * (int64_t)M_pad;
  const int stage = mx_outer_stage<T>(job.rows), part_bytes = min(kMxOuterRows, job.rows) * kMxOuterTokens * 2;
  constexpr uint32_t kTopsAt = kMxOuterXBytes, kPartsAt = kTopsAt + kMxOuterTops;
  const uint32_t a_at = kPartsAt + ar * 64 + ((threadIdx.x & 3) << 4);
  // f16: 16 exponents of a group, by the first threads
  const bool tops = HALF && (int)threadIdx.x < 2 * groups;
  const int tgroup = (int)threadIdx.x >= groups, tpiece = (int)threadIdx.x - (tgroup ? groups : 0);
  const uint8_t* tp = job.tops + (int64_t)(2 * s0 + tgroup) * job.rows + row0 + 16 * tpiece;
  int m_next = s0 * kMxOuterTokens + tok;
  const int m_end = s1 * kMxOuterTokens;  // (tok < 8: a step begins before it or not at all)
  MxRing in, out;
  auto fetch = [&]() {
    if (m_next < m_end) {
      const uint32_t base = smem_u32(mx_smem) + in.at * stage;
      const T* x = xp;
#pragma unroll
      for (int u = 0; u < 4; ++u, x += x_eight) {
        const bool here = m_next + 8 * u < M;
        cp_async16(base + x_at[u], here ? x : job.X, here ? bytes : 0);
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        if (ar < rows) cp_async16(base + a_at + part * part_bytes, ap + part * part_off, 16);
        if (ar + 32 < rows) cp_async16(base + a_at + part * part_bytes + 32 * 64, ap + part * part_off + row32, 16);
      }
      if (tops) cp_async16(base + kTopsAt + tgroup * kMxOuterRows + 16 * tpiece, tp, 16);
      xp += 4 * x_eight;
      ap += kMxOuterTokens;
      tp += 2 * (int64_t)job.rows;
      m_next += kMxOuterTokens;
      in.next(kMxOuterStages);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k < kMxOuterStages - 1; ++k) fetch();

  __shared__ int row_top[HALF ? kMxOuterRows : 1];  // the rows' largest exponents among this CTA's tokens
  if constexpr (HALF) {
    if (threadIdx.x < kMxOuterRows) row_top[threadIdx.x] = 0;
    __syncthreads();
    const int row = threadIdx.x & (kMxOuterRows - 1);
    int top = 0;
    if (row < rows)
      for (int k = 2 * s0 + (int)(threadIdx.x / kMxOuterRows); k < 2 * s1; k += 128 / kMxOuterRows)
        top = max(top, (int)__ldcg(job.tops + (int64_t)k * job.rows + row0 + row));
    atomicMax(&row_top[row], top);  // a maximum: the same in any order
    __syncthreads();
  }

  float acc[4][4][4] = {};  // [row group][8 columns][fragment]
  float sum[4] = {};
  const bool sums = job.sums && rt == 0;
  // this lane's row of the transposing loads: matrix lane / 8 (pair j), row lane % 8
  const int mtok = 8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1);
  const int mf = (mtok & 1) | ((mtok >> 3) & 3) << 1;
  for (int step = s0; step < s1; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kMxOuterStages - 2) : "memory");
    __syncthreads();
    fetch();  // into the stage of the step before: every warp is past it
    const uint32_t base = smem_u32(mx_smem) + out.at * stage;
    out.next(kMxOuterStages);
    uint32_t b[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                   : "=r"(b[n][0]), "=r"(b[n][1]), "=r"(b[n][2]), "=r"(b[n][3])
                   : "r"(base + mtok * 256 + (((4 * warp + n) ^ mf) << 4))
                   : "memory");
    if (sums) {  // the lane holds eight tokens of column g
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[n] += HALF ? __low2float(*reinterpret_cast<const __half2*>(&b[n][j])) +
                               __high2float(*reinterpret_cast<const __half2*>(&b[n][j]))
                         : __uint_as_float(b[n][j] << 16) + __uint_as_float(b[n][j] & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < groups) {
        uint32_t fl = 0u, fh = 0u;  // f16: of rows g and g + 8, this lane's eight tokens
        if constexpr (HALF) {
          const uint8_t* at = mx_smem + (base - smem_u32(mx_smem)) + kTopsAt + (t >> 1) * kMxOuterRows + 16 * r + g;
          fl = mx_top_factor(at[0], row_top[16 * r + g]);
          fh = mx_top_factor(at[8], row_top[16 * r + g + 8]);
        }
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const uint32_t at = base + kPartsAt + part * part_bytes + (16 * r + g) * 64 + t * 16;
          uint4 l = lds128(at), h = lds128(at + 8 * 64);
          if constexpr (HALF) {
            l.x = mx_mul2<true>(l.x, fl); l.y = mx_mul2<true>(l.y, fl);
            l.z = mx_mul2<true>(l.z, fl); l.w = mx_mul2<true>(l.w, fl);
            h.x = mx_mul2<true>(h.x, fh); h.y = mx_mul2<true>(h.y, fh);
            h.z = mx_mul2<true>(h.z, fh); h.w = mx_mul2<true>(h.w, fh);
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            mx_mma<HALF>(acc[r][n], l.x, h.x, l.y, h.y, b[n][0], b[n][1]);
            mx_mma<HALF>(acc[r][n], l.z, h.z, l.w, h.w, b[n][2], b[n][3]);
          }
        }
      }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < groups) {
      float down[2] = {1.f, 1.f};  // of rows g and g + 8
      if constexpr (HALF) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int top = row_top[16 * r + g + 8 * h];
          if (top) down[h] = scalbnf(1.f, top - 141);  // 1 / mx_top_scale
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = row0 + 16 * r + g + 8 * (q >> 1), c = c0 + 32 * warp + 8 * n + 2 * t + (q & 1);
          if (c < job.cols) job.partial[((int64_t)split * job.rows + row) * job.cols + c] = acc[r][n][q] * down[q >> 1];
        }
    }
  if (sums)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float v = sum[n];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int c = c0 + 32 * warp + 8 * n + g;
      if (t == 0 && c < job.cols) job.sums[(int64_t)split * job.cols + c] = v;
    }
  if (beside && blockIdx.x == gridDim.x - 1) pdl_wait_prior();
}

// ---------------------------------------------------------------------------
// fp32: on the CUDA cores
// ---------------------------------------------------------------------------
constexpr int kMxOuter32Cols = 128;   // columns of a CTA, one per thread
constexpr int kMxOuter32Ranks = 32;   // ranks of a CTA, in registers
constexpr int kMxOuter32Tokens = 32;  // tokens whose t is staged at a time

// partial[split][r][c] = sum_m t[m, r] X[m, c] (and the column sums of X).
__global__ void __launch_bounds__(kMxOuter32Cols)
qlin_mx_outer32_kernel(const __grid_constant__ MxOuterJob<float> job0, const __grid_constant__ MxOuterJob<float> job1,
                       int M) {
  __shared__ float4 ts[kMxOuter32Tokens][kMxOuter32Ranks / 4];
  pdl_wait_prior();
  pdl_launch_dependents();
  const bool first = (int)blockIdx.x < job0.blocks;
  const MxOuterJob<float>& job = first ? job0 : job1;
  int id = (int)blockIdx.x - (first ? 0 : job0.blocks);
  const int ct = id % job.col_tiles;
  id /= job.col_tiles;
  const int rt = id % job.row_tiles, split = id / job.row_tiles;
  const int m0 = (int)((int64_t)M * split / job.splits), m1 = (int)((int64_t)M * (split + 1) / job.splits);
  const int c = ct * kMxOuter32Cols + threadIdx.x, r0 = rt * kMxOuter32Ranks;
  const bool here = c < job.cols;
  const float* x = job.X + (here ? c : 0);
  float4 acc[kMxOuter32Ranks / 4];
#pragma unroll
  for (int r = 0; r < kMxOuter32Ranks / 4; ++r) acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int m = m0; m < m1; m += kMxOuter32Tokens) {
    __syncthreads();
    for (int k = threadIdx.x; k < kMxOuter32Tokens * kMxOuter32Ranks; k += kMxOuter32Cols) {
      const int tok = k / kMxOuter32Ranks, r = r0 + k % kMxOuter32Ranks;
      reinterpret_cast<float*>(ts)[k] =
          m + tok < m1 && r < job.rows ? __ldcg(job.turned + (int64_t)(m + tok) * job.rows + r) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int u0 = 0; u0 < kMxOuter32Tokens; u0 += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = m + u0 + u < m1 ? __ldcg(x + (int64_t)(m + u0 + u) * job.ld) : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        sum += v[u];
#pragma unroll
        for (int r = 0; r < kMxOuter32Ranks / 4; ++r) {
          const float4 t = ts[u0 + u][r];
          acc[r].x = fmaf(t.x, v[u], acc[r].x);
          acc[r].y = fmaf(t.y, v[u], acc[r].y);
          acc[r].z = fmaf(t.z, v[u], acc[r].z);
          acc[r].w = fmaf(t.w, v[u], acc[r].w);
        }
      }
    }
  }
  if (!here) return;
#pragma unroll
  for (int r = 0; r < kMxOuter32Ranks; ++r)
    if (r0 + r < job.rows)
      job.partial[((int64_t)split * job.rows + r0 + r) * job.cols + c] = reinterpret_cast<const float*>(acc)[r];
  if (job.sums && rt == 0) job.sums[(int64_t)split * job.cols + c] = sum;
}

// Adds the splits up: da [rank, cols] from job0's; db [cols, rank] and dbias
// [cols] from job1's.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_outer_finish_kernel(const __grid_constant__ MxOuterJob<T> job0, const __grid_constant__ MxOuterJob<T> job1,
                            int rank, T* da, T* db, T* dbias, int64_t blocks0) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const bool first = (int64_t)blockIdx.x < blocks0;
  const MxOuterJob<T>& job = first ? job0 : job1;
  const int64_t k = ((int64_t)blockIdx.x - (first ? 0 : blocks0)) * 256 + threadIdx.x;
  const int rows = first ? rank : rank + (dbias ? 1 : 0);
  if (k >= (int64_t)rows * job.cols) return;
  // consecutive threads: consecutive columns of a row
  const int64_t r = k / job.cols, c = k - r * job.cols;
  const bool bias = r == rank;
  const float* at = bias ? job.sums + c : job.partial + r * job.cols + c;
  const int64_t step = bias ? job.cols : (int64_t)job.rows * job.cols;
  float v = 0.f;
  for (int s = 0; s < job.splits; ++s) v += __ldcg(at + s * step);
  if (first) da[k] = from_f32<T>(v);
  else if (bias) dbias[c] = from_f32<T>(v);
  else db[c * rank + r] = from_f32<T>(v);
}

}  // namespace qlin
