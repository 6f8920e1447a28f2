// Global norm of many gradient tensors, and their clipping:
//
//     norm = sqrt(sum over all tensors and elements of g^2)
//     g   <- g * min(1, max_norm / (norm + 1e-6))
//
// Two launches over one table of tensors (a kernel parameter: no copy to the
// device, so both can be captured into a graph).  The elements of all tensors
// form one line of pieces of kClipPiece elements, no piece in two tensors; the
// CTAs take batches of kClipBatch pieces in turn, so that at any time they read
// one stretch of the line.
//
// Bound by the bytes: read once for the norm, read and written once for the
// product.  The second launch walks the line backwards, so that it begins with
// what the first has left in L2; a set that L2 holds is read from HBM once.
// 48 bf16 gradients, 270 MB: 136 us (4.0 TB/s if only one read and the write count;
// three passes at HBM's rate: 124 us).  48 fp32 gradients of adapters, 25 MB, which L2
// holds: 17 us.
// (Evict-first hints for all but the last 40 or 72 MB of the first pass changed
// nothing: 134 to 142 us for 270 MB either way.)
//
// Squares are summed in fp32 within a piece and thread (8 terms) and in fp64 from
// there on, in an order that depends only on the sizes: the same gradients give
// the same bits.  A thread whose fp32 sum overflows, or is so small that squares may
// have been lost below fp32's numbers (2^-90, or zero), sums its piece again in fp64.
#pragma once

#include "qlin_common.cuh"

namespace qlin {

constexpr int kClipThreads = 256;
constexpr int kClipEach = 8;                          // elements of a thread
constexpr int kClipPiece = kClipThreads * kClipEach;  // elements
constexpr int kClipBatch = 4;                         // whole pieces of a tensor whose loads go out together
constexpr int kClipTensors = 512;              // most table entries of a launch
constexpr int kClipFewTensors = 64;            // entries of the small table (less to hand to a launch)
constexpr int kClipCtasPerSm = 6;

template <int CAP>
struct ClipTable {
  void* data[CAP];
  long long first[CAP + 1];  // first piece of each tensor
  long long size[CAP];       // elements
  unsigned char type[CAP];   // QLIN_F32, QLIN_BF16, QLIN_F16
  int count;
};

// A thread's elements of a whole, aligned piece: 16-byte pieces apart by
// kClipThreads * 16 bytes.
template <typename T>
struct ClipLoad {
  static constexpr int V = 16 / (int)sizeof(T);
  uint4 q[kClipEach / V];
  __device__ __forceinline__ void load(const T* piece) {
#pragma unroll
    for (int u = 0; u < kClipEach / V; ++u) q[u] = ld_cg_v4(piece + (u * kClipThreads + threadIdx.x) * V);
  }
  __device__ __forceinline__ double squares() const {
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < kClipEach / V; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float v = to_f32(reinterpret_cast<const T*>(&q[u])[j]);
        s = fmaf(v, v, s);
      }
    if (s >= 0x1p-90f && s <= 3.0e38f) return (double)s;
    double d = 0.0;
#pragma unroll
    for (int u = 0; u < kClipEach / V; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double v = (double)to_f32(reinterpret_cast<const T*>(&q[u])[j]);
        d += v * v;
      }
    return d;
  }
  __device__ __forceinline__ void store_scaled(T* piece, float f) {
#pragma unroll
    for (int u = 0; u < kClipEach / V; ++u) {
      T* e = reinterpret_cast<T*>(&q[u]);
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = from_f32<T>(to_f32(e[j]) * f);
      *reinterpret_cast<uint4*>(piece + (u * kClipThreads + threadIdx.x) * V) = q[u];
    }
  }
};

// The sum of squares of this thread's elements of `n` consecutive pieces of a
// tensor, of which `left` elements are there.
template <typename T>
__device__ __forceinline__ double clip_sum(const T* at, int n, long long left) {
  double d = 0.0;
  if ((reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    if (n == kClipBatch && left >= (long long)kClipBatch * kClipPiece) {
      ClipLoad<T> a[kClipBatch];
#pragma unroll
      for (int u = 0; u < kClipBatch; ++u) a[u].load(at + u * kClipPiece);
#pragma unroll
      for (int u = 0; u < kClipBatch; ++u) d += a[u].squares();
      return d;
    }
    for (; n > 0 && left >= kClipPiece; --n, left -= kClipPiece, at += kClipPiece) {
      ClipLoad<T> a;
      a.load(at);
      d += a.squares();
    }
  }
  const long long rest = min(left, (long long)n * kClipPiece);
  for (long long k = threadIdx.x; k < rest; k += kClipThreads) {
    const double v = (double)to_f32(at[k]);
    d += v * v;
  }
  return d;
}

template <typename T>
__device__ __forceinline__ void clip_scale(T* at, int n, long long left, float f) {
  if ((reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    if (n == kClipBatch && left >= (long long)kClipBatch * kClipPiece) {
      ClipLoad<T> a[kClipBatch];
#pragma unroll
      for (int u = 0; u < kClipBatch; ++u) a[u].load(at + u * kClipPiece);
#pragma unroll
      for (int u = 0; u < kClipBatch; ++u) a[u].store_scaled(at + u * kClipPiece, f);
      return;
    }
    for (; n > 0 && left >= kClipPiece; --n, left -= kClipPiece, at += kClipPiece) {
      ClipLoad<T> a;
      a.load(at);
      a.store_scaled(at, f);
    }
  }
  const long long rest = min(left, (long long)n * kClipPiece);
  for (long long k = threadIdx.x; k < rest; k += kClipThreads) at[k] = from_f32<T>(to_f32(at[k]) * f);
}

// Sum of all threads' values, the same in every thread (fixed order).
__device__ __forceinline__ double clip_block_sum(double v, double* slots) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 32; ++w) s += slots[w];
  return s;
}

// partials[blockIdx.x] = this CTA's share of the sum of squares.
template <int CAP>
__global__ void __launch_bounds__(kClipThreads, kClipCtasPerSm)
qlin_grad_norm_kernel(const __grid_constant__ ClipTable<CAP> tab, double* partials) {
  __shared__ double slots[kClipThreads / 32];
  pdl_wait_prior();
  pdl_launch_dependents();
  const long long pieces = tab.first[tab.count];
  double s = 0.0;
  int k = 0;
  for (long long b = (long long)blockIdx.x * kClipBatch; b < pieces; b += (long long)gridDim.x * kClipBatch) {
    for (long long p = b; p < min(pieces, b + kClipBatch);) {
      while (p >= tab.first[k + 1]) ++k;
      const int n = (int)(min(b + kClipBatch, tab.first[k + 1]) - p);
      const long long at = (p - tab.first[k]) * kClipPiece, left = tab.size[k] - at;
      if (tab.type[k] == 0) s += clip_sum(static_cast<const float*>(tab.data[k]) + at, n, left);
      else if (tab.type[k] == 1) s += clip_sum(static_cast<const __nv_bfloat16*>(tab.data[k]) + at, n, left);
      else s += clip_sum(static_cast<const __half*>(tab.data[k]) + at, n, left);
      p += n;
    }
  }
  s = clip_block_sum(s, slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// Every CTA adds up all partial sums (in the same order) and scales its pieces.
template <int CAP>
__global__ void __launch_bounds__(kClipThreads, kClipCtasPerSm)
qlin_grad_scale_kernel(const __grid_constant__ ClipTable<CAP> tab, const double* partials, int n_partials,
                       float max_norm, float* norm_out) {
  __shared__ double slots[kClipThreads / 32];
  pdl_wait_prior();
  pdl_launch_dependents();
  double s = 0.0;
  for (int k = threadIdx.x; k < n_partials; k += kClipThreads) s += __ldcg(partials + k);
  s = clip_block_sum(s, slots);
  const float norm = (float)sqrt(s);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  // a NaN norm makes every gradient NaN, an infinite one zero (or NaN)
  float f = max_norm / (norm + 1e-6f);
  if (f > 1.f) f = 1.f;
  if (isinf(max_norm)) return;  // the norm alone
  const long long pieces = tab.first[tab.count], batches = (pieces + kClipBatch - 1) / kClipBatch;
  int k = tab.count - 1;
  for (long long b = batches - 1 - blockIdx.x; b >= 0; b -= gridDim.x) {  // backwards
    for (long long p = min(pieces, (b + 1) * kClipBatch); p > b * kClipBatch;) {
      while (p - 1 < tab.first[k]) --k;
      const int n = (int)(p - max(b * kClipBatch, tab.first[k]));
      p -= n;
      const long long at = (p - tab.first[k]) * kClipPiece, left = tab.size[k] - at;
      if (tab.type[k] == 0) clip_scale(static_cast<float*>(tab.data[k]) + at, n, left, f);
      else if (tab.type[k] == 1) clip_scale(static_cast<__nv_bfloat16*>(tab.data[k]) + at, n, left, f);
      else clip_scale(static_cast<__half*>(tab.data[k]) + at, n, left, f);
    }
  }
}

}  // namespace qlin
