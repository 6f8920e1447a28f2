// The adapter's products in the backward pass of a layer with 4-bit weights.
//
//     t  = s x A^T          [M, r]      t' = s gy B           [M, r]
//     dA = t'^T x           [r, K]      dB = gy^T t           [N, r]
//     dbias = sum_m gy[m]   [N]
//
// t and t' stay in fp32: rounded to 16 bits they would add an error of the
// size of the gradients' own rounding.
#pragma once

#include "qlin_common.cuh"

namespace qlin {

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

// dst[c][r] = src[r][c]
template <typename T>
__global__ void __launch_bounds__(256)
qlin_mx_turn_kernel(const T* __restrict__ src, T* __restrict__ dst, int64_t rows, int64_t cols) {
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (k < rows * cols) dst[(k % cols) * rows + k / cols] = src[k];
}

}  // namespace qlin
