// The adapter's products around a layer with 4-bit weights.
//
//     t  = s x A^T          [M, r]      u  = s gy B           [M, r]
//     dA = u^T x            [r, K]      dB = gy^T t           [N, r]
//     dbias = sum_m gy[m]   [N]
//
// t and u are kept as two 16-bit parts (or in fp32): rounded to one they would
// add an error of the size of the gradients' own rounding.  x and gy are read
// once for t and u and once for the gradients, which bounds these kernels; the
// products are warp-level tensor-core ones (m16n8k16) whose k slots are numbered
// so that a lane reads eight consecutive elements of a row in one 16-byte piece
// for both operands.
#pragma once

#include "qlin_common.cuh"
#include "qlin_mx_few.cuh"

namespace qlin {

// ---------------------------------------------------------------------------
// fp32: plain products
// ---------------------------------------------------------------------------
// C[i, j] = alpha * sum_l P[i pi + l pl] * Q[j qj + l ql], fp32 sums; C is
// row-major with leading dimension ld_c.  32 x 32 tile, 32 terms per step.
template <typename TP, typename TQ, typename TC>
__global__ void __launch_bounds__(256)
qlin_mx_strided_gemm_kernel(const TP* __restrict__ P, int64_t pi, int64_t pl, const TQ* __restrict__ Q, int64_t qj,
                            int64_t ql, TC* __restrict__ C, int64_t ld_c, int64_t I, int64_t J, int64_t L,
                            float alpha) {
  __shared__ float ps[32][33], qs[32][33];
  const int64_t i0 = (int64_t)blockIdx.x * 32, j0 = (int64_t)blockIdx.y * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float acc[4] = {};
  for (int64_t l0 = 0; l0 < L; l0 += 32) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // lanes along the contiguous direction of each operand
      const int s = ty + 8 * u;
      const int pr = pl == 1 ? s : tx, pc = pl == 1 ? tx : s;
      const int qr = ql == 1 ? s : tx, qc = ql == 1 ? tx : s;
      ps[pr][pc] = i0 + pr < I && l0 + pc < L ? to_f32(P[(i0 + pr) * pi + (l0 + pc) * pl]) : 0.f;
      qs[qr][qc] = j0 + qr < J && l0 + qc < L ? to_f32(Q[(j0 + qr) * qj + (l0 + qc) * ql]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int l = 0; l < 32; ++l) {
      const float q = qs[tx][l];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = fmaf(ps[ty + 8 * u][l], q, acc[u]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = i0 + ty + 8 * u, j = j0 + tx;
    if (i < I && j < J) C[i * ld_c + j] = from_f32<TC>(alpha * acc[u]);
  }
}

// out[n] = sum_m g[m, n]
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_column_sum_kernel(const T* __restrict__ g, int64_t ld_g, T* __restrict__ out, int64_t M, int64_t N) {
  __shared__ float part[8][32];
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

// dst[c][r] = src[r][c] for two matrices.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_turn_kernel(const T* __restrict__ a, T* __restrict__ at, int64_t a_rows, int64_t a_cols,
                    const T* __restrict__ b, T* __restrict__ bt, int64_t b_rows, int64_t b_cols, int64_t a_blocks) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const bool first = (int64_t)blockIdx.x < a_blocks;
  const int64_t k = ((int64_t)blockIdx.x - (first ? 0 : a_blocks)) * 256 + threadIdx.x;
  const int64_t rows = first ? a_rows : b_rows, cols = first ? a_cols : b_cols;
  // consecutive threads write consecutive elements
  if (k < rows * cols) (first ? at : bt)[k] = (first ? a : b)[(k % rows) * cols + k / rows];
}

constexpr int kMxTurnRows = 64;  // output quaternions of a step

// What the 16-bit gradients need turned, in one launch: blocks [0, steps) make
// the components of conj(W)^T 2^-c (rows of ld elements), the next a_blocks A^T,
// the rest B^T.  A step is 64 output x 32 input quaternions; a thread takes two
// neighbouring output quaternions, eight input quaternions and two components,
// so that the turned pairs go to shared memory as words, a warp's in a row.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_turn_all_kernel(const uint8_t* __restrict__ mx, const MxPlanes<T> dst, int64_t ld, int K_g, int N_g,
                        int64_t steps, const T* __restrict__ a, T* __restrict__ at, int64_t a_rows, int64_t a_cols,
                        const T* __restrict__ b, T* __restrict__ bt, int64_t b_rows, int64_t b_cols,
                        int64_t a_blocks) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  __shared__ __align__(16) uint32_t turned[4 * kMxBlock][36];  // [component, input quaternion][pair of outputs]
  pdl_wait_prior();
  pdl_launch_dependents();
  if ((int64_t)blockIdx.x >= steps) {
    const bool first = (int64_t)blockIdx.x < steps + a_blocks;
    const int64_t k = ((int64_t)blockIdx.x - steps - (first ? 0 : a_blocks)) * 256 + threadIdx.x;
    const int64_t rows = first ? a_rows : b_rows, cols = first ? a_cols : b_cols;
    // consecutive threads write consecutive elements
    if (k < rows * cols) (first ? at : bt)[k] = (first ? a : b)[(k % rows) * cols + k / rows];
    return;
  }
  const int64_t kb = (K_g + kMxBlock - 1) / kMxBlock, tiles = (N_g + kMxRows - 1) / kMxRows;
  const int64_t og = blockIdx.x / kb, blk = blockIdx.x - og * kb;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = warp & 3, ph = warp >> 2;
  uint32_t f0;
  asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(f0) : "l"(mx) : "memory");
  const int c = mx_shift<HALF>(f0, a_rows > 0 ? 1 : 0);
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
    for (int u = 0; u < 2; ++u)
      mx_expand_scaled<HALF>(pw, h ? w[u].y : w[u].x,
                             mx_multiplier<HALF>((f[u] >> (8 * h)) & 255u, c) ^ (p ? 0x80008000u : 0u), e[u]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      turned[p * kMxBlock + 8 * t + k][lane] = __byte_perm(e[0][k], e[1][k], 0x5410);
      turned[p * kMxBlock + 8 * t + k + 4][lane] = __byte_perm(e[0][k], e[1][k], 0x7632);
    }
  }
  __syncthreads();
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

// dst rows of ld_d elements (ld_d >= cols), zero past cols: rows that no TMA map takes.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_repack_kernel(const T* __restrict__ src, int64_t ld_s, T* __restrict__ dst, int64_t ld_d, int64_t rows,
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

template <typename T>
struct MxDownJob {
  const T* x;      // [M, ld_x], 16-byte aligned rows
  int64_t ld_x;
  const T* a;      // [rank, K]
  int64_t K;
  float scale;
  T* parts;        // [M, 2, ld_parts]: hi and lo, zero from rank to ld_parts; or null
  T* turned;       // [2][rows][M_pad]: hi, then lo, transposed; or null
  int rank, ld_parts, rows, vec;  // vec: rows of A are 16-byte aligned
  int rank_tiles;  // ceil(max(ld_parts, rows) / 32)
  int blocks;
};

// Eight elements of a row of K, zero past its end.
template <typename T>
__device__ __forceinline__ uint4 mx_load_row8(const T* row, int64_t k, int64_t K, bool vec) {
  if (vec && k + 8 <= K) return ld_cg_v4(row + k);
  unsigned short h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    h[j] = k + j < K ? *reinterpret_cast<const volatile unsigned short*>(row + k + j) : (unsigned short)0;
  return make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                    h[6] | (uint32_t)h[7] << 16);
}

// A CTA: 16 tokens x 32 ranks, its eight warps every eighth piece of 32 terms.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_down_kernel(const __grid_constant__ MxDownJob<T> job0, const __grid_constant__ MxDownJob<T> job1, int M, int M_pad) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  __shared__ float red[8][kMxDownRows][kMxDownRanks + 1];
  pdl_wait_prior();
  pdl_launch_dependents();
  const bool first = (int)blockIdx.x < job0.blocks;
  const MxDownJob<T>& job = first ? job0 : job1;
  const int id = (int)blockIdx.x - (first ? 0 : job0.blocks);
  const int m0 = id / job.rank_tiles * kMxDownRows, r0 = id % job.rank_tiles * kMxDownRanks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float acc[4][4] = {};
  const T* xl = job.x + (int64_t)(m0 + g) * job.ld_x;
  const T* xh = xl + 8 * job.ld_x;
  const bool has_l = m0 + g < M, has_h = m0 + g + 8 < M;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  // four pieces at a time: 24 loads of 16 bytes in flight per lane
  for (int64_t k0 = 32 * warp; k0 < job.K && r0 < job.rank; k0 += 4 * 32 * 8) {
    uint4 lo[4], hi[4], b[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t k = k0 + u * 32 * 8 + 8 * t;
      const bool in = k < job.K;
      lo[u] = in && has_l ? mx_load_row8(xl, k, job.K, true) : zero;
      hi[u] = in && has_h ? mx_load_row8(xh, k, job.K, true) : zero;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = r0 + 8 * n + g;
        b[u][n] = in && r < job.rank ? mx_load_row8(job.a + (int64_t)r * job.K, k, job.K, job.vec) : zero;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        mx_mma<HALF>(acc[n], lo[u].x, hi[u].x, lo[u].y, hi[u].y, b[u][n].x, b[u][n].y);
        mx_mma<HALF>(acc[n], lo[u].z, hi[u].z, lo[u].w, hi[u].w, b[u][n].z, b[u][n].w);
      }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) red[warp][g + 8 * (q >> 1)][8 * n + 2 * t + (q & 1)] = acc[n][q];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    // hi and lo of (token, rank); ranks fastest for `parts`, tokens fastest for `turned`
#pragma unroll
    for (int way = 0; way < 2; ++way) {
      if (way == 0 ? !job.parts : !job.turned) continue;
      const int k = threadIdx.x + 256 * u;
      const int m = way == 0 ? k >> 5 : k & 15, r = way == 0 ? k & 31 : k >> 4;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += red[w][m][r];
      v *= job.scale;
      const T hi = from_f32<T>(v);
      const float rest = v - to_f32(hi);
      const T lo = from_f32<T>(isfinite(rest) ? rest : 0.f);  // (hi infinite or NaN: alone)
      if (way == 0) {
        if (m0 + m < M && r0 + r < job.ld_parts) {
          T* at = job.parts + (int64_t)(m0 + m) * 2 * job.ld_parts + r0 + r;
          at[0] = hi;
          at[job.ld_parts] = lo;
        }
      } else if (r0 + r < job.rows) {
        T* at = job.turned + (int64_t)(r0 + r) * M_pad + m0 + m;
        at[0] = hi;
        at[(int64_t)job.rows * M_pad] = lo;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit gradients: out = (hi + lo) X, sums over the tokens
// ---------------------------------------------------------------------------
constexpr int kMxOuterCols = 128;   // columns of X of a CTA, 16 per warp
constexpr int kMxOuterTokens = 32;  // tokens of a step
constexpr int kMxOuterRows = 64;    // rows of the result of a CTA (groups of 16)
constexpr int kMxOuterStages = 4;
constexpr int kMxOuterXBytes = kMxOuterTokens * kMxOuterCols * 2;
constexpr int kMxOuterStage = kMxOuterXBytes + 2 * kMxOuterRows * kMxOuterTokens * 2;
constexpr int kMxOuterSmem = kMxOuterStages * kMxOuterStage;

template <typename T>
struct MxOuterJob {
  const T* turned;  // [2][rows][M_pad]
  const T* X;       // [M, ld], 16-byte aligned rows
  int64_t ld;
  int cols, rows;   // rows: a multiple of 16
  int col_tiles, row_tiles, splits;
  int blocks;
  float* partial;   // [splits][rows][cols]
  float* sums;      // [splits][cols] column sums of X, or null
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Eight warps: 16 columns each, all rows.  X and the rows of (hi, lo) come through
// a ring of shared memory steps (32 tokens x 128 columns; 16-byte chunks permuted
// within a row of X so that the transposing loads of eight tokens two apart are
// free of conflicts).
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_outer_kernel(const __grid_constant__ MxOuterJob<T> job0, const __grid_constant__ MxOuterJob<T> job1, int M,
                     int M_pad) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t mx_smem[];
  pdl_wait_prior();
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
  const T* turned = job.turned + (int64_t)row0 * M_pad;
  const int64_t lo_off = (int64_t)job.rows * M_pad;

  auto fetch = [&](int step) {
    if (step < s1) {
      const uint32_t base = smem_u32(mx_smem) + (step % kMxOuterStages) * kMxOuterStage;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = threadIdx.x + 256 * u, tok = k >> 4, chunk = k & 15;
        const int m = step * kMxOuterTokens + tok, c = c0 + 8 * chunk;
        const int left = m < M ? min(8, job.cols - c) : 0;  // elements of the chunk inside
        const int f = (tok & 1) | ((tok >> 3) & 3) << 1;
        cp_async16(base + tok * 256 + ((chunk ^ f) << 4), left > 0 ? job.X + (int64_t)m * job.ld + c : job.X,
                   left > 0 ? 2 * left : 0);
      }
      for (int k = threadIdx.x; k < 8 * rows; k += 256) {  // [part][row][4 chunks]
        const int part = k >= 4 * rows ? 1 : 0, r = (k - part * 4 * rows) >> 2, chunk = k & 3;
        cp_async16(base + kMxOuterXBytes + (part * kMxOuterRows + r) * 64 + (chunk << 4),
                   turned + part * lo_off + (int64_t)r * M_pad + step * kMxOuterTokens + 8 * chunk, 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k < kMxOuterStages - 1; ++k) fetch(s0 + k);

  float acc[4][2][4] = {};  // [row group][8 columns][fragment]
  float sum[2] = {0.f, 0.f};
  const bool sums = job.sums && rt == 0;
  // this lane's row of the transposing loads: matrix lane / 8 (pair j), row lane % 8
  const int mtok = 8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1);
  const int mf = (mtok & 1) | ((mtok >> 3) & 3) << 1;
  for (int step = s0; step < s1; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kMxOuterStages - 2) : "memory");
    __syncthreads();
    fetch(step + kMxOuterStages - 1);  // into the stage of step - 1: every warp is past it
    const uint32_t base = smem_u32(mx_smem) + (step % kMxOuterStages) * kMxOuterStage;
    uint32_t b[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                   : "=r"(b[n][0]), "=r"(b[n][1]), "=r"(b[n][2]), "=r"(b[n][3])
                   : "r"(base + mtok * 256 + (((2 * warp + n) ^ mf) << 4))
                   : "memory");
    if (sums) {  // the lane holds eight tokens of column g
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const T* e = reinterpret_cast<const T*>(&b[n][j]);
          sum[n] += to_f32(e[0]) + to_f32(e[1]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < groups)
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const uint32_t at = base + kMxOuterXBytes + (part * kMxOuterRows + 16 * r + g) * 64 + t * 16;
          const uint4 l = lds128(at), h = lds128(at + 8 * 64);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            mx_mma<HALF>(acc[r][n], l.x, h.x, l.y, h.y, b[n][0], b[n][1]);
            mx_mma<HALF>(acc[r][n], l.z, h.z, l.w, h.w, b[n][2], b[n][3]);
          }
        }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < groups)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = row0 + 16 * r + g + 8 * (q >> 1), c = c0 + 16 * warp + 8 * n + 2 * t + (q & 1);
          if (c < job.cols) job.partial[((int64_t)split * job.rows + row) * job.cols + c] = acc[r][n][q];
        }
  if (sums)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float v = sum[n];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int c = c0 + 16 * warp + 8 * n + g;
      if (t == 0 && c < job.cols) job.sums[(int64_t)split * job.cols + c] = v;
    }
}

// Adds the splits up: da [rank, cols] from job0's; db [cols, rank] and dbias
// [cols] from job1's.
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_outer_finish_kernel(const __grid_constant__ MxOuterJob<T> job0, const __grid_constant__ MxOuterJob<T> job1, int rank, T* __restrict__ da,
                            T* __restrict__ db, T* __restrict__ dbias, int64_t blocks0) {
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
