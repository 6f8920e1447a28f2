// C ABI of the 4-bit (MXFP4) quaternion weights and of gradient clipping
// (declarations: include/qlin_b200.h): argument checks, workspace pieces,
// launches on the caller's stream.  No exception crosses the ABI, nothing
// allocates.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "../../include/qlin_b200.h"
#include "qlin_clip.cuh"
#include "qlin_host.h"
#include "qlin_mx.cuh"
#include "qlin_mx_few.cuh"
#include "qlin_mx_lora.cuh"
#include "qlin_mx_pair.cuh"

namespace {

using namespace qlin;

inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline bool known(int dtype) { return dtype == QLIN_F32 || dtype == QLIN_BF16 || dtype == QLIN_F16; }
inline int64_t elem(int dtype) { return dtype == QLIN_F32 ? 4 : 2; }

int check_groups(int64_t K_g, int64_t N_g) {
  if (K_g <= 0 || N_g <= 0 || K_g > INT32_MAX / 8 || N_g > INT32_MAX / 8) return QLIN_ERR_SHAPE;
  return QLIN_OK;
}

int64_t mx_bytes(int64_t K_g, int64_t N_g) {
  return kMxHeader + ceil_div(N_g, kMxRows) * ceil_div(K_g, kMxBlock) * kMxRecord;
}

// Tokens and ranks whose padded counts and tiles stay within 32 bits.
constexpr int64_t kMostTokens = INT32_MAX - 1023;
constexpr int kMostRanks = 1 << 24;

int check_layer(int dtype, int64_t M, int64_t K_g, int64_t N_g, int rank) {
  if (!known(dtype)) return QLIN_ERR_DTYPE;
  if (M < 0 || M > kMostTokens || rank < 0 || rank > kMostRanks) return QLIN_ERR_SHAPE;
  return check_groups(K_g, N_g);
}

int launched() { return cudaGetLastError() == cudaSuccess ? QLIN_OK : QLIN_ERR_LAUNCH; }

// Calls f(element value of the type) for a known dtype.
template <typename F>
int by_type(int dtype, F f) {
  switch (dtype) {
    case QLIN_F32: return f(float());
    case QLIN_BF16: return f(__nv_bfloat16());
    default: return f(__half());
  }
}

// Pieces of a workspace, 256-byte aligned.
struct Carve {
  size_t at = 0;
  size_t take(int64_t bytes) {
    const size_t p = at;
    at = (size_t)round_up((int64_t)at + bytes, 256);
    return p;
  }
};

// SM count that the rules below reckon with: they size workspaces, which do not depend
// on the device.  (Launches take the device's own.)
constexpr int64_t kRuleSms = 148;

// 16-bit inputs of up to 32 tokens take the streaming kernels (qlin_mx_few.cuh; 5120 ->
// 27648 at 32 tokens 39 against 47 us), and up to 64 where the layer has at most a tile
// of 16 output quaternions per SM (4096 -> 4096 at 64 tokens 13 against 21 us, 5120 ->
// 27648 70 against 47); more take the CTA-pair kernel (qlin_mx_pair.cuh).  fp32 always
// streams.
bool streams(int dtype, int64_t M, int64_t N_g) {
  return dtype == QLIN_F32 || M <= 32 || (M <= 64 && N_g <= kRuleSms * kMxRows);
}

// Tokens of a tile of the streaming kernels (one or two tokens apart).  16 bits: two
// tiles of 16 run beside each other faster than one of 32 (4096 -> 4096 at 32 tokens
// 9.3 against 12.7 us, 11008 -> 4096 16.8 against 22.2), three or four do not (64
// tokens 17.7 against 12.9).  fp32, which comes here with any number of tokens: 16
// (by two tiles of output quaternions) or 32 (by four) by the waves of CTAs, of which
// one of 32 takes as long as about 3.5 of 16 (4096 -> 11008 at 128 tokens 108 against
// 150 us, 768 -> 2304 at 512 tokens 37 against 30).
int few_tile(int dtype, int64_t M, int64_t N_g) {
  if (M <= 16) return M <= 8 ? 8 : 16;
  if (dtype != QLIN_F32) return M <= 32 ? 16 : 32;
  const int64_t waves16 = ceil_div(ceil_div(N_g, 2 * kMxRows) * ceil_div(M, 16), kRuleSms);
  const int64_t waves32 = ceil_div(ceil_div(N_g, 4 * kMxRows) * ceil_div(M, 32), kRuleSms);
  return 2 * waves16 <= 7 * waves32 ? 16 : 32;
}

// One or two tokens whose B words fit beside a ring of two stages of 16 warps and
// everything else that a CTA of theirs may hold.
constexpr size_t kMostSmem = 226 * 1024;  // 1 KB of the 227 left for static shared memory
constexpr size_t kOneMaxX = 148 * 1024;
static_assert(kOneMaxX + 2 * (16 * kMxRecord + 16) + 2 * 16 * 2 * kMxRedRow * 4 + kMxMostB + 2 * kMxSmemRank * 4 + 64 <=
                  kMostSmem,
              "a layer that is_one() admits has to fit");
bool is_one(int dtype, int64_t M, int64_t K_g) {
  const int64_t kb = ceil_div(K_g, kMxBlock);
  return M <= 2 && (size_t)kb * 1024 * (dtype == QLIN_F32 ? 3 : 1) + M * 4 * K_g * elem(dtype) <= kOneMaxX;
}

// Rows of 16-bit elements that TMA takes: 16-byte aligned start and row stride.
bool tma_rows(const void* p, int64_t ld) { return aligned(p, 16) && ld % 8 == 0; }

int64_t pair_parts(int dtype) { return dtype == QLIN_F16 ? kMxPairParts<__half> : kMxPairParts<__nv_bfloat16>; }

struct ForwardWs {
  size_t arranged = 0, t = 0, x = 0, a = 0, total = 0;
  int64_t ld_parts = 0;  // ranks of t's rows, in whole 16-byte pieces
};

// Sized for the worst alignment of x: the pieces do not depend on pointers.
ForwardWs forward_ws(int dtype, int64_t M, int64_t K_g, int64_t N_g, int rank) {
  ForwardWs w;
  Carve c;
  if (streams(dtype, M, N_g)) {
    if (!is_one(dtype, M, K_g)) {
      const int64_t C = few_tile(dtype, M, N_g);
      w.arranged = c.take(ceil_div(M, C) * ceil_div(K_g, kMxBlock) * (dtype == QLIN_F32 ? 3 : 1) * 4 * C * 64);
    }
    w.t = c.take(M * rank * 4);
  } else {
    w.ld_parts = round_up(rank, 8);
    w.x = c.take(M * round_up(4 * K_g, 8) * 2);
    w.t = c.take(M * pair_parts(dtype) * w.ld_parts * 2);
    w.a = c.take(rank * round_up(4 * K_g, 8) * 2);
  }
  w.total = c.at;
  return w;
}

struct BackwardWs {
  // (fp32: planes are wide records, gy its B words)
  size_t gy = 0, x = 0, a = 0, at = 0, bt = 0, parts = 0, up = 0, t = 0, planes = 0, partial0 = 0, partial1 = 0, sums = 0,
         up_tops = 0, t_tops = 0;
  int64_t M_pad = 0, ld_parts = 0, ld_planes = 0;
  int rows = 0, splits0 = 0, splits1 = 0;
  size_t total = 0;
};

// Splits of the tokens of a gradient product: about two CTAs per SM for each of the
// two (three fit an SM; short ones fill more of what the input gradient's last wave
// leaves free: 4096 layer at 2048 tokens, forward and gradients 141 us in a graph, 143
// with 1.5), at least four steps of 32 tokens each.
int outer_splits(int64_t M_pad, int64_t cols, int rows) {
  const int64_t tiles = ceil_div(cols, kMxOuterCols) * ceil_div(rows, kMxOuterRows);
  return (int)std::max<int64_t>(1, std::min<int64_t>(M_pad / kMxOuterTokens / 4, 320 / std::max<int64_t>(1, tiles)));
}

// The same for fp32: about two CTAs per SM each, at least 32 tokens.
int outer32_splits(int64_t M, int64_t cols, int rank) {
  const int64_t tiles = ceil_div(cols, kMxOuter32Cols) * ceil_div(rank, kMxOuter32Ranks);
  return (int)std::max<int64_t>(1, std::min<int64_t>(M / 32, 296 / std::max<int64_t>(1, tiles)));
}

BackwardWs backward_ws(int dtype, int64_t M, int64_t K_g, int64_t N_g, int rank) {
  BackwardWs w;
  Carve c;
  if (dtype == QLIN_F32) {
    const int64_t C = few_tile(dtype, M, K_g);
    w.planes = c.take(ceil_div(K_g, kMxRows) * ceil_div(N_g, kMxBlock) * kMxWideRecord);
    w.gy = c.take(ceil_div(M, C) * ceil_div(N_g, kMxBlock) * 3 * 4 * C * 64);
    if (rank > 0) {
      w.at = c.take(4 * K_g * rank * 4);
      w.splits0 = outer32_splits(M, 4 * K_g, rank);
      w.splits1 = outer32_splits(M, 4 * N_g, rank);
      w.bt = c.take(4 * N_g * rank * 4);
      w.t = c.take(M * rank * 4);
      w.up = c.take(M * rank * 4);
      w.partial0 = c.take((int64_t)w.splits0 * rank * 4 * K_g * 4);
      w.partial1 = c.take((int64_t)w.splits1 * rank * 4 * N_g * 4);
      w.sums = c.take((int64_t)w.splits1 * 4 * N_g * 4);
    }
  } else {
    const int64_t K = 4 * K_g, N = 4 * N_g;
    w.M_pad = round_up(M, kMxOuterTokens);
    w.ld_parts = round_up(rank, 8);
    w.ld_planes = round_up(N_g, 8);
    w.rows = (int)round_up(rank, 16);
    w.splits0 = outer_splits(w.M_pad, K, w.rows);
    w.splits1 = outer_splits(w.M_pad, N, w.rows);
    w.gy = c.take(M * round_up(N, 8) * 2);
    w.x = c.take(rank > 0 ? M * round_up(K, 8) * 2 : 0);
    w.planes = c.take(4 * K_g * w.ld_planes * 2);
    if (rank > 0) {
      w.at = c.take(K * rank * 2);
      w.bt = c.take(round_up(N, 8) * rank * 2);
      w.a = c.take(rank * round_up(K, 8) * 2);
      w.parts = c.take(M * pair_parts(dtype) * w.ld_parts * 2);
      const int64_t parts = dtype == QLIN_F16 ? kMxTurnedParts<__half> : kMxTurnedParts<__nv_bfloat16>;
      w.up = c.take(parts * w.rows * w.M_pad * 2);
      w.t = c.take(parts * w.rows * w.M_pad * 2);
      if (dtype == QLIN_F16) {
        w.up_tops = c.take(w.M_pad / kMxDownRows * w.rows);
        w.t_tops = c.take(w.M_pad / kMxDownRows * w.rows);
      }
      w.partial0 = c.take((int64_t)w.splits0 * w.rows * K * 4);
      w.partial1 = c.take((int64_t)w.splits1 * w.rows * N * 4);
      w.sums = c.take((int64_t)w.splits1 * N * 4);
    }
  }
  w.total = c.at;
  return w;
}

// Grid of the record kernels: a warp takes four rows (y) of two records (x) at a
// time; about `ctas` CTAs.
dim3 record_grid(int64_t K_g, int64_t N_g, int64_t ctas) {
  const int64_t rows = ceil_div(N_g, kMxRows) * (kMxRows / kMxUnitRows), x = ceil_div(K_g, 2 * kMxBlock * 8);
  return dim3((unsigned)x, (unsigned)std::min<int64_t>({rows, ceil_div(ctas, x), 32768}));
}

template <typename T>
void launch_dequantize(const void* mx, const MxPlanes<T>& dst, int64_t ld, int64_t K_g, int64_t N_g,
                       cudaStream_t s) {
  bool vec = (ld * sizeof(T)) % 16 == 0;
  for (int c = 0; c < 4; ++c) vec = vec && aligned(dst.w[c], 16);
  qlin_mx_dequantize_kernel<T><<<record_grid(K_g, N_g, INT32_MAX), 256, 0, s>>>(static_cast<const uint8_t*>(mx), dst, ld,
                                                                         (int)K_g, (int)N_g, vec);
}

// Launch as a programmatic dependent of the stream's previous kernel.
template <typename... KArgs, typename... Args>
int launch_dependent(void (*kernel)(KArgs...), unsigned ctas, unsigned threads, size_t smem, cudaStream_t s,
                     Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
}

// Raises a kernel's shared-memory limit once per device.
template <typename K>
int allow_smem(K kernel, std::atomic<uint64_t>& done, size_t bytes = kMostSmem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return QLIN_ERR_LAUNCH;
  if (done.load(std::memory_order_acquire) >> dev & 1) return QLIN_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
    return QLIN_ERR_LAUNCH;
  done.fetch_or(1ull << dev, std::memory_order_release);
  return QLIN_OK;
}

// Stages of a ring: what fits `budget` beside `fixed` bytes, at least 2, at
// most what a CTA uses.
int ring_stages(size_t budget, size_t fixed, size_t stage, int64_t uses) {
  const int64_t fit = budget > fixed ? (int64_t)((budget - fixed) / stage) : 0;
  return (int)std::max<int64_t>(2, std::min(fit, uses));
}

// Pieces that rows of lora_b are made of (16 or 8 bytes, or 0), and whether a CTA keeps
// those of a tile of 64 `wo` outputs in shared memory.
template <typename T>
int pieces_b(const MxFewParams<T>& prm) {
  for (const int piece : {16, 8})
    if (prm.rank > 0 && prm.rank * sizeof(T) % piece == 0 && aligned(prm.lora_b, piece)) return piece;
  return 0;
}
template <typename T>
bool stages_b(const MxFewParams<T>& prm, int wo) {
  return pieces_b(prm) == 16 && prm.rank <= kMxSmemRank && mx_b_bytes<T>(prm.rank, wo) <= kMxMostB;
}

// W warps per tile, G tiles of a CTA at a time; QLIN_ERR_SHAPE where that does not fit.
template <typename T, int W, int G>
int launch_one(const MxFewParams<T>& base, int sms, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  MxFewParams<T> prm = base;
  const int ctas = (int)std::min<int64_t>(prm.tiles, sms);
  const int64_t uses = ceil_div(prm.kb, W) * ceil_div(prm.tiles, (int64_t)ctas * G);
  prm.stage_b = stages_b(prm, 1);
  prm.vec_b = pieces_b(prm);
  const int b = prm.stage_b ? mx_b_bytes<T>(prm.rank, 1) : 0;
  prm.ring = ring_stages(kMostSmem, mx_one_smem<T, W, G>(prm.M, prm.K_g, 0, prm.rank, b), G * (W * kMxRecord + 16),
                         uses);
  const size_t smem = mx_one_smem<T, W, G>(prm.M, prm.K_g, prm.ring, prm.rank, b);
  if (smem > kMostSmem) return QLIN_ERR_SHAPE;
  if (allow_smem(qlin_mx_one_kernel<T, W, G>, done) != QLIN_OK) return QLIN_ERR_LAUNCH;
  return launch_dependent(qlin_mx_one_kernel<T, W, G>, ctas, 32 * (W + 1) * G, smem, s, prm);
}

template <typename T, int NT, int WO, bool WIDE = false>
int launch_many(const MxFewParams<T>& base, int sms, cudaStream_t s) {
  using Cfg = MxManyCfg<T, NT, WO, WIDE>;
  static std::atomic<uint64_t> done{0};
  if (allow_smem(qlin_mx_many_kernel<T, NT, WO, WIDE>, done) != QLIN_OK) return QLIN_ERR_LAUNCH;
  MxFewParams<T> prm = base;
  const int64_t total = ceil_div(prm.tiles, WO) * ceil_div(prm.M, Cfg::kC);
  prm.stage_b = stages_b(prm, WO);
  prm.vec_b = pieces_b(prm);
  const int b = prm.stage_b ? mx_b_bytes<T>(prm.rank, WO) : 0;
  const size_t fixed = mx_many_smem<T, NT, WO, WIDE>(0, prm.rank, b), stage = Cfg::kStage + 16;
  // two CTAs per SM (tiles of 8 tokens, whose registers allow it) where their rings fit
  // and the last wave stays as full (8 tokens, 4096 -> 11008: 172 tiles, 10.3 against
  // 11.8 us; 5120 -> 27648: 432 tiles, 18.3 against 17.0)
  constexpr size_t kHalfSm = kMostSmem / 2 - 1024;
  const bool two = NT == 1 && sizeof(T) == 2 && total > sms && 2 * ceil_div(total, 2 * sms) <= ceil_div(total, sms) &&
                   fixed + 2 * stage <= kHalfSm;
  const int ctas = (int)std::min<int64_t>(total, (two ? 2 : 1) * sms);
  const int64_t uses = ceil_div(prm.kb, Cfg::kWK) * ceil_div(total, ctas);
  prm.ring = ring_stages(two ? kHalfSm : kMostSmem, fixed, stage, uses);
  const size_t smem = mx_many_smem<T, NT, WO, WIDE>(prm.ring, prm.rank, b);
  if (smem > kMostSmem) return QLIN_ERR_SHAPE;
  return launch_dependent(qlin_mx_many_kernel<T, NT, WO, WIDE>, ctas, kMxThreads, smem, s, prm);
}

// The B words of x (none for `one`) and the scaled down projection, in the workspace.
template <typename T>
int few_prologue(const MxFewParams<T>& prm, bool one, const T* a, float scale, uint8_t* arranged, float* t,
                 cudaStream_t s) {
  const int C = few_tile(sizeof(T) == 4 ? QLIN_F32 : QLIN_BF16, prm.M, prm.N_g);
  const int64_t token_groups = ceil_div(prm.M, kMxDownTokens);
  const bool ranks = prm.rank * token_groups >= 4 * 222;  // 1.5 CTAs of four ranks per SM
  const int threads = ranks ? 256 : mx_prologue_threads(prm.K_g);
  const int64_t octets = one ? 0 : ceil_div(prm.M, C) * C * 4 * prm.kb;
  const int64_t blocks = ceil_div(octets, threads), down = (ranks ? ceil_div(prm.rank, kMxDownRanksMost) : prm.rank) * token_groups;
  if (blocks + down > INT32_MAX) return QLIN_ERR_SHAPE;
  if (blocks + down == 0) return QLIN_OK;
  const int vec = aligned(prm.x, 4 * sizeof(T)) && prm.ld_x % 4 == 0;
  return launch_dependent(ranks ? qlin_mx_prologue_kernel<T, kMxDownRanksMost> : qlin_mx_prologue_kernel<T, 1>,
                          (unsigned)(blocks + down), threads, 0, s, prm.x, prm.ld_x, prm.M,
                          prm.K_g, prm.kb, C, vec, arranged, (int)blocks, octets, a,
                          (int)aligned(a, 4 * sizeof(T)), prm.rank, scale, t);
}

// The streaming kernels: a prologue where there are B words to arrange or an
// adapter, then the product.
template <typename T>
int run_few(int dtype, const T* x, int64_t ld_x, const void* mx, const T* bias, const T* a, const T* b, int rank,
            float scale, T* y, int64_t ld_y, int64_t M, int64_t K_g, int64_t N_g, uint8_t* ws, const ForwardWs& w,
            int sms, cudaStream_t s) {
  MxFewParams<T> prm{};
  prm.x = x;
  prm.ld_x = ld_x;
  prm.mx = static_cast<const uint8_t*>(mx);
  prm.records = prm.mx + kMxHeader;
  prm.arranged = ws + w.arranged;
  prm.bias = bias;
  prm.lora_b = b;
  prm.t = reinterpret_cast<const float*>(ws + w.t);
  prm.y = y;
  prm.ld_y = ld_y;
  prm.M = (int)M;
  prm.K_g = (int)K_g;
  prm.N_g = (int)N_g;
  prm.rank = rank;
  prm.kb = (int)ceil_div(K_g, kMxBlock);
  prm.tiles = (int)ceil_div(N_g, kMxRows);
  const bool one = is_one(dtype, M, K_g);
  const int C = few_tile(dtype, M, N_g);
  const int st = few_prologue(prm, one, a, scale, ws + w.arranged, reinterpret_cast<float*>(ws + w.t), s);
  if (st != QLIN_OK) return st;
  if (one) {
    prm.after_prologue = rank > 0;
    // x by bulk copies
    prm.vec = aligned(x, 16) && (4 * K_g * sizeof(T)) % 16 == 0 && (M == 1 || (ld_x * sizeof(T)) % 16 == 0);
    // at most a tile per SM, or x too long for three rings: 16 warps share the
    // tile's K (4096 -> 4096: 4.2 against 4.6 us); more tiles: three groups of 8 warps
    // (5120 -> 27648: 8.3 against 8.8 us, graph replays)
    if (prm.tiles > sms) {
      const int e = launch_one<T, 8, 3>(prm, sms, s);
      if (e != QLIN_ERR_SHAPE) return e;
    }
    return launch_one<T, 16, 1>(prm, sms, s);
  }
  if (C == 8) return launch_many<T, 1, 1>(prm, sms, s);
  // Side by side, tiles of a CTA share the B words (two or four of them: fp32's are
  // too long for one); alone, there are more CTAs.  16 bits at 16 tokens: a wave of two
  // side by side takes as long as 1.4 waves of one, so side by side where that halves
  // the waves (4096 -> 11008: 2 waves -> 1, 17.1 -> 12.8 us; 5120 -> 27648: 3 against
  // 2, 24.7 against 29.0).  Tiles of 32 tokens come with few tiles.
  if constexpr (sizeof(T) == 2) {
    if (C == 32) return launch_many<T, 4, 1>(prm, sms, s);
    const int64_t alone = ceil_div(prm.tiles * ceil_div(M, C), sms);
    const int64_t beside = ceil_div(ceil_div(prm.tiles, 2) * ceil_div(M, C), sms);
    return alone < 2 * beside ? launch_many<T, 2, 1>(prm, sms, s) : launch_many<T, 2, 2>(prm, sms, s);
  } else {
    return C == 16 ? launch_many<T, 2, 2>(prm, sms, s) : launch_many<T, 4, 4>(prm, sms, s);
  }
}

// ---------------------------------------------------------------------------
// many tokens, 16 bits
// ---------------------------------------------------------------------------
// A TMA map of `dims` (innermost first; `strides` in elements from the second on).
int encode_map(CUtensorMap* map, bool bf16, const void* base, int rank, const int64_t (&dims)[3],
               const int64_t (&strides)[2], const uint32_t (&box)[3], CUtensorMapSwizzle swizzle) {
  const auto encode = qlin_host_encoder();
  if (!encode) return QLIN_ERR_LAUNCH;
  const cuuint64_t d[3] = {(cuuint64_t)dims[0], (cuuint64_t)dims[1], (cuuint64_t)dims[2]};
  const cuuint64_t st[2] = {(cuuint64_t)(strides[0] * 2), (cuuint64_t)(strides[1] * 2)};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank,
                const_cast<void*>(base), d, st, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? QLIN_OK
             : QLIN_ERR_ALIGN;
}

// How many CTA pairs of a kernel the device holds at once (0: not known).
template <typename T, int NTOK, bool MX>
int pair_capacity() {
  auto kernel = qlin_mx_pair_kernel<T, NTOK, MX>;
  constexpr size_t smem = kPairSmemBytes;
  static std::mutex mutex;
  static int capacity[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(mutex);
  if (capacity[dev] == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2, 1, 1);
    cfg.blockDim = dim3(kMxPairThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute a;
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = 2;
    a.val.clusterDim.y = 1;
    a.val.clusterDim.z = 1;
    cfg.attrs = &a;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 0;
    }
    capacity[dev] = n;
  }
  return capacity[dev];
}

// y = x W^T (+ bias) (+ parts B^T) on the CTA-pair kernel: W from codes (mx) or
// from component planes.  x rows satisfy tma_rows; y 8-byte aligned, ld_y a
// multiple of 4.  With an adapter the launch before it is the down projection that
// makes `parts`.
template <typename T, int NTOK, bool MX>
int launch_pair(const T* x, int64_t ld_x, const void* mx, const MxPlanes<T>& planes, int64_t ld_w, const T* bias,
                const __nv_bfloat16* parts, int64_t ld_parts, const T* lora_b, int rank, T* y, int64_t ld_y, int64_t M,
                int64_t K_g, int64_t N_g, cudaStream_t s) {
  using Cfg = MxPairStage<NTOK, MX>;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  auto kernel = qlin_mx_pair_kernel<T, NTOK, MX>;
  const int cap = pair_capacity<T, NTOK, MX>();
  if (cap == 0) return QLIN_ERR_LAUNCH;
  CUtensorMap map_x, map_t, map_w[4];
  std::memset(&map_t, 0, sizeof(map_t));
  std::memset(map_w, 0, sizeof(map_w));
  int st = encode_map(&map_x, bf16, x, 2, {4 * K_g, M, 1}, {ld_x, 0}, {64, Cfg::kHalf, 1}, CU_TENSOR_MAP_SWIZZLE_128B);
  const int64_t terms = kMxPairParts<T> * ld_parts;
  if (st == QLIN_OK && rank > 0)  // [token][term]: past the last term zero
    st = encode_map(&map_t, true, parts, 2, {terms, M, 1}, {terms, 0}, {64, Cfg::kHalf, 1}, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!MX)
    for (int p = 0; p < 4 && st == QLIN_OK; ++p)
      st = encode_map(&map_w[p], bf16, planes.w[p], 2, {K_g, N_g, 1}, {ld_w, 0}, {32, 32, 1}, CU_TENSOR_MAP_SWIZZLE_64B);
  if (st != QLIN_OK) return st;
  MxPairParams prm{};
  prm.mx = static_cast<const uint8_t*>(mx);
  prm.bias = bias;
  prm.lora_b = lora_b;
  prm.y = y;
  prm.ld_y = ld_y;
  prm.M = (int)M;
  prm.N_g = (int)N_g;
  prm.K_g = (int)K_g;
  prm.rank = rank;
  prm.kb = (int)ceil_div(K_g, kMxBlock);
  prm.w_tiles = (int)ceil_div(N_g, kMxRows);
  prm.stages = (int)ceil_div(K_g, 32);
  prm.ld_parts = (int)ld_parts;
  prm.lora_stages = rank > 0 ? (int)ceil_div(ld_parts, kMxPairRanks<T>) : 0;
  prm.nb_tiles = (int)ceil_div(4 * N_g, 256);
  const int64_t tiles = prm.nb_tiles * ceil_div(M, NTOK);
  if (tiles * (prm.stages + prm.lora_stages) > INT32_MAX) return QLIN_ERR_SHAPE;
  prm.tiles = (int)tiles;
  prm.wide = aligned(y, 16) && ld_y % 8 == 0 && N_g % 2 == 0;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = 2;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, cap)), 1, 1);
  cfg.blockDim = dim3(kMxPairThreads, 1, 1);
  cfg.dynamicSmemBytes = kPairSmemBytes;
  cfg.stream = s;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, map_x, map_t, map_w[0], map_w[1], map_w[2], map_w[3], prm) == cudaSuccess
             ? QLIN_OK
             : QLIN_ERR_LAUNCH;
}

// Tiles of 256 tokens, or of 128 where those end sooner: a wave of them takes nearly
// 0.8 of the time (stages of 0.55 us, the expansion's time, against 0.71), and few
// tokens or outputs leave pairs without a tile of 256.  (256 -> 128: 4096 -> 4096 at
// 256 tokens, 1 wave each, 27.4 -> 21.6 us; 4096 -> 11008 at 512 tokens, 2 against 3
// waves, 47.8 -> 55.9.)
template <typename T, bool MX, typename... Args>
int run_pair(int64_t M, int64_t N_g, Args... args) {
  const int64_t nb = ceil_div(4 * N_g, 256), cap = std::max(1, pair_capacity<T, 256, MX>());
  const int64_t waves256 = ceil_div(nb * ceil_div(M, 256), cap), waves128 = ceil_div(nb * ceil_div(M, 128), cap);
  return 9 * waves128 < 11 * waves256 ? launch_pair<T, 128, MX>(args...) : launch_pair<T, 256, MX>(args...);
}

// Rows that TMA takes (whole: and that are whole 16-byte pieces): x itself, or a
// copy in the workspace with zeros up to the next 16 bytes.
template <typename T>
int rows_for_tma(const T** x, int64_t* ld, void* copy, int64_t rows, int64_t cols, bool whole, cudaStream_t s) {
  if (tma_rows(*x, *ld) && !(whole && cols % 8 != 0)) return QLIN_OK;
  const int64_t ld_c = round_up(cols, 8), blocks = ceil_div(rows * ld_c, 256);
  if (blocks > INT32_MAX) return QLIN_ERR_SHAPE;
  const int st = launch_dependent(qlin_mx_repack_kernel<T>, (unsigned)blocks, 256, 0, s, *x, *ld, static_cast<T*>(copy),
                                  ld_c, rows, cols);
  *x = static_cast<const T*>(copy);
  *ld = ld_c;
  return st;
}

template <typename T>
MxDownJob<T> down_job(const T* x, int64_t ld_x, const T* a, int64_t ld_a, int64_t K, float scale, int rank,
                      __nv_bfloat16* parts, int64_t ld_parts, T* turned, uint8_t* tops, int rows, int64_t tokens) {
  MxDownJob<T> j{};
  j.x = x;
  j.ld_x = ld_x;
  j.a = a;
  j.ld_a = ld_a;
  j.K = (int)round_up(K, 8);
  j.scale = scale;
  j.rank = rank;
  j.parts = parts;
  j.ld_parts = parts ? (int)ld_parts : 0;
  j.turned = turned;
  j.tops = tops;
  j.rows = turned ? rows : 0;
  j.rank_tiles = (int)ceil_div(std::max(j.ld_parts, j.rows), kMxDownRanks);
  j.blocks = (int)(ceil_div(tokens, kMxDownRows) * j.rank_tiles);
  return j;
}

template <typename T>
int launch_down(const MxDownJob<T>& j0, const MxDownJob<T>& j1, int64_t M, int64_t M_pad, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  if (allow_smem(qlin_mx_down_kernel<T>, done, kMxDownSmem) != QLIN_OK) return QLIN_ERR_LAUNCH;
  return launch_dependent(qlin_mx_down_kernel<T>, (unsigned)(j0.blocks + j1.blocks), 256, kMxDownSmem, s, j0, j1,
                          (int)M, (int)M_pad);
}

template <typename T>
int run_prefill(const T* x, int64_t ld_x, const void* mx, const T* bias, const T* a, const T* b, int rank, float scale,
                T* y, int64_t ld_y, int64_t M, int64_t K_g, int64_t N_g, uint8_t* ws, const ForwardWs& w,
                cudaStream_t s) {
  if (!aligned(y, 8) || ld_y % 4 != 0) return QLIN_ERR_ALIGN;
  int st = rows_for_tma(&x, &ld_x, ws + w.x, M, 4 * K_g, rank > 0, s);
  if (st != QLIN_OK) return st;
  __nv_bfloat16* parts = reinterpret_cast<__nv_bfloat16*>(ws + w.t);
  if (rank > 0) {
    int64_t ld_a = 4 * K_g;
    st = rows_for_tma(&a, &ld_a, ws + w.a, rank, 4 * K_g, true, s);
    if (st != QLIN_OK) return st;
    const MxDownJob<T> job = down_job<T>(x, ld_x, a, ld_a, 4 * K_g, scale, rank, parts, w.ld_parts, nullptr, nullptr, 0, M);
    st = launch_down<T>(job, MxDownJob<T>{}, M, M, s);
    if (st != QLIN_OK) return st;
  }
  return run_pair<T, true>(M, N_g, x, ld_x, mx, MxPlanes<T>{}, (int64_t)0, bias, (const __nv_bfloat16*)parts,
                           w.ld_parts, b, rank, y, ld_y, M, K_g, N_g, s);
}

// Gradients, 16 bits.
template <typename T>
int run_backward(const T* g, int64_t ld_g, const T* x, int64_t ld_x, const void* mx, const T* a, const T* b, int rank,
                 float scale, T* dx, int64_t ld_dx, T* da, T* db, T* dbias, int64_t M, int64_t K_g, int64_t N_g,
                 uint8_t* ws, const BackwardWs& w, cudaStream_t s) {
  const int64_t K = 4 * K_g, N = 4 * N_g;
  if (dx && (!aligned(dx, 8) || ld_dx % 4 != 0)) return QLIN_ERR_ALIGN;
  T* at = reinterpret_cast<T*>(ws + w.at);
  T* bt = reinterpret_cast<T*>(ws + w.bt);
  __nv_bfloat16* parts = reinterpret_cast<__nv_bfloat16*>(ws + w.parts);
  T* up = reinterpret_cast<T*>(ws + w.up);
  T* t = reinterpret_cast<T*>(ws + w.t);
  int st = QLIN_OK;
  if (dx || da || db) st = rows_for_tma(&g, &ld_g, ws + w.gy, M, N, rank > 0, s);
  if (st == QLIN_OK && (da || db)) st = rows_for_tma(&x, &ld_x, ws + w.x, M, K, true, s);
  const T* a8 = a;  // A's rows, in whole 16-byte pieces
  int64_t ld_a = K;
  if (st == QLIN_OK && db) st = rows_for_tma(&a8, &ld_a, ws + w.a, rank, K, true, s);
  if (st != QLIN_OK) return st;
  const bool need_up = rank > 0 && (dx || da);
  MxPlanes<T> p{};
  if (dx || need_up) {
    // conj(W)^T, A^T and B^T
    for (int c = 0; c < 4; ++c) p.w[c] = reinterpret_cast<T*>(ws + w.planes) + c * K_g * w.ld_planes;
    const int64_t steps = dx ? ceil_div(N_g, kMxTurnRows) * ceil_div(K_g, kMxBlock) : 0;
    const int64_t a_blocks = dx ? ceil_div(rank * K, 256) : 0, b_blocks = need_up ? ceil_div(rank * round_up(N, 8), 256) : 0;
    if (steps + a_blocks + b_blocks > INT32_MAX) return QLIN_ERR_SHAPE;
    st = launch_dependent(qlin_mx_turn_all_kernel<T>, (unsigned)(steps + a_blocks + b_blocks), 256, 0, s,
                          static_cast<const uint8_t*>(mx), p, w.ld_planes, (int)K_g, (int)N_g, steps, a, at,
                          (int64_t)rank, K, b, bt, N, (int64_t)rank, round_up(N, 8), a_blocks);
    if (st != QLIN_OK) return st;
  }
  if (rank > 0 && (need_up || db)) {
    MxDownJob<T> j0{}, j1{};
    if (need_up)
      j0 = down_job<T>(g, ld_g, bt, round_up(N, 8), N, scale, rank, dx ? parts : nullptr, w.ld_parts,
                       da ? up : nullptr, ws + w.up_tops, w.rows, w.M_pad);
    if (db)
      j1 = down_job<T>(x, ld_x, a8, ld_a, K, scale, rank, nullptr, 0, t, ws + w.t_tops, w.rows, w.M_pad);
    st = launch_down<T>(j0, j1, M, w.M_pad, s);
    if (st != QLIN_OK) return st;
  }
  if (dx) {
    st = run_pair<T, false>(M, K_g, g, ld_g, mx, p, w.ld_planes, (const T*)nullptr, (const __nv_bfloat16*)parts,
                            w.ld_parts, (const T*)at, rank, dx, ld_dx, M, N_g, K_g, s);
    if (st != QLIN_OK) return st;
  }
  const bool sum_with_db = db && dbias;
  if (da || db) {
    MxOuterJob<T> o0{}, o1{};
    auto job = [&](MxOuterJob<T>& o, const T* turned, size_t tops, const T* X, int64_t ld, int64_t cols, int rows,
                   int splits, size_t partial) {
      o.turned = turned;
      o.tops = ws + tops;
      o.X = X;
      o.ld = ld;
      o.cols = (int)cols;
      o.rows = rows;
      o.col_tiles = (int)ceil_div(cols, kMxOuterCols);
      o.row_tiles = (int)ceil_div(rows, kMxOuterRows);
      o.splits = splits;
      o.blocks = o.col_tiles * o.row_tiles * splits;
      o.partial = reinterpret_cast<float*>(ws + partial);
    };
    if (da) job(o0, up, w.up_tops, x, ld_x, K, w.rows, w.splits0, w.partial0);
    if (db) job(o1, t, w.t_tops, g, ld_g, N, w.rows, w.splits1, w.partial1);
    static std::atomic<uint64_t> done{0};
    if (allow_smem(qlin_mx_outer_kernel<T>, done, kMxOuterStages * mx_outer_stage<T>(kMxOuterRows)) != QLIN_OK)
      return QLIN_ERR_LAUNCH;
    if (sum_with_db) o1.sums = reinterpret_cast<float*>(ws + w.sums);
    st = launch_dependent(qlin_mx_outer_kernel<T>, (unsigned)(o0.blocks + o1.blocks), 128,
                          kMxOuterStages * mx_outer_stage<T>(w.rows), s, o0, o1,
                          (int)M, (int)w.M_pad, (int)(dx != nullptr));
    if (st != QLIN_OK) return st;
    const int64_t blocks0 = da ? ceil_div(rank * K, 256) : 0;
    const int64_t blocks1 = db ? ceil_div((rank + (sum_with_db ? 1 : 0)) * N, 256) : 0;
    st = launch_dependent(qlin_mx_outer_finish_kernel<T>, (unsigned)(blocks0 + blocks1), 256, 0, s, o0, o1, rank, da,
                          db, sum_with_db ? dbias : nullptr, blocks0);
    if (st != QLIN_OK) return st;
  }
  if (dbias && !sum_with_db)
    st = launch_dependent(qlin_mx_column_sum_kernel<T>, (unsigned)ceil_div(N, 32), 256, 0, s, g, ld_g, dbias, M, N);
  return st != QLIN_OK ? st : launched();
}

// Gradients, fp32: dx by the streaming kernel on the adjoint's wide records, the
// adapter's on the CUDA cores.
int run_backward32(const float* g, int64_t ld_g, const float* x, int64_t ld_x, const void* mx, const float* a,
                   const float* b, int rank, float scale, float* dx, int64_t ld_dx, float* da, float* db, float* dbias,
                   int64_t M, int64_t K_g, int64_t N_g, uint8_t* ws, const BackwardWs& w, int sms, cudaStream_t s) {
  const int64_t K = 4 * K_g, N = 4 * N_g;
  float* at = reinterpret_cast<float*>(ws + w.at);
  float* bt = reinterpret_cast<float*>(ws + w.bt);
  float* t = reinterpret_cast<float*>(ws + w.t);
  float* up = reinterpret_cast<float*>(ws + w.up);
  uint8_t* arranged = ws + w.gy;
  const bool need_up = rank > 0 && (dx || da);
  int st = QLIN_OK;
  if (dx || need_up) {
    MxPlanes<float> records{};
    records.w[0] = reinterpret_cast<float*>(ws + w.planes);
    const int64_t steps = dx ? ceil_div(N_g, kMxTurnRows) * ceil_div(K_g, kMxBlock) : 0;
    const int64_t a_blocks = dx ? ceil_div(rank * K, 256) : 0, b_blocks = need_up ? ceil_div(rank * N, 256) : 0;
    if (steps + a_blocks + b_blocks > INT32_MAX) return QLIN_ERR_SHAPE;
    st = launch_dependent(qlin_mx_turn_all_kernel<float>, (unsigned)(steps + a_blocks + b_blocks), 256, 0, s,
                          static_cast<const uint8_t*>(mx), records, (int64_t)0, (int)K_g, (int)N_g, steps, a, at,
                          (int64_t)rank, K, b, bt, N, (int64_t)rank, N, a_blocks);
    if (st != QLIN_OK) return st;
    MxFewParams<float> prm{};
    prm.x = g;
    prm.ld_x = ld_g;
    prm.mx = static_cast<const uint8_t*>(mx);
    prm.records = ws + w.planes;
    prm.arranged = arranged;
    prm.lora_b = at;
    prm.t = up;
    prm.y = dx;
    prm.ld_y = ld_dx;
    prm.M = (int)M;
    prm.K_g = (int)N_g;
    prm.N_g = (int)K_g;
    prm.rank = rank;
    prm.kb = (int)ceil_div(N_g, kMxBlock);
    prm.tiles = (int)ceil_div(K_g, kMxRows);
    st = few_prologue(prm, !dx, (const float*)bt, scale, arranged, up, s);
    if (st != QLIN_OK) return st;
    if (dx) {
      const int C = few_tile(QLIN_F32, M, K_g);
      st = C == 8 ? launch_many<float, 1, 1, true>(prm, sms, s)
                  : (C == 16 ? launch_many<float, 2, 2, true>(prm, sms, s) : launch_many<float, 4, 4, true>(prm, sms, s));
      if (st != QLIN_OK) return st;
    }
  }
  if (db) {
    MxFewParams<float> prm{};
    prm.x = x;
    prm.ld_x = ld_x;
    prm.M = (int)M;
    prm.K_g = (int)K_g;
    prm.rank = rank;
    st = few_prologue(prm, true, a, scale, static_cast<uint8_t*>(nullptr), t, s);
    if (st != QLIN_OK) return st;
  }
  const bool sum_with_db = db && dbias;
  if (da || db) {
    MxOuterJob<float> o0{}, o1{};
    auto job = [&](MxOuterJob<float>& o, const float* rows, const float* X, int64_t ld, int64_t cols, int splits,
                   size_t partial) {
      o.turned = rows;
      o.X = X;
      o.ld = ld;
      o.cols = (int)cols;
      o.rows = rank;
      o.col_tiles = (int)ceil_div(cols, kMxOuter32Cols);
      o.row_tiles = (int)ceil_div(rank, kMxOuter32Ranks);
      o.splits = splits;
      o.blocks = o.col_tiles * o.row_tiles * splits;
      o.partial = reinterpret_cast<float*>(ws + partial);
    };
    if (da) job(o0, up, x, ld_x, K, w.splits0, w.partial0);
    if (db) job(o1, t, g, ld_g, N, w.splits1, w.partial1);
    if (sum_with_db) o1.sums = reinterpret_cast<float*>(ws + w.sums);
    st = launch_dependent(qlin_mx_outer32_kernel, (unsigned)(o0.blocks + o1.blocks), kMxOuter32Cols, 0, s, o0, o1,
                          (int)M);
    if (st != QLIN_OK) return st;
    const int64_t blocks0 = da ? ceil_div(rank * K, 256) : 0;
    const int64_t blocks1 = db ? ceil_div((rank + (sum_with_db ? 1 : 0)) * N, 256) : 0;
    st = launch_dependent(qlin_mx_outer_finish_kernel<float>, (unsigned)(blocks0 + blocks1), 256, 0, s, o0, o1, rank,
                          da, db, sum_with_db ? dbias : nullptr, blocks0);
    if (st != QLIN_OK) return st;
  }
  if (dbias && !sum_with_db)
    st = launch_dependent(qlin_mx_column_sum_kernel<float>, (unsigned)ceil_div(N, 32), 256, 0, s, g, ld_g, dbias, M, N);
  return st != QLIN_OK ? st : launched();
}

template <int CAP>
void clip_tables(int count, void* const* grads, const int64_t* sizes, const int* dtypes, float max_norm, float* norm,
                 double* partials, int ctas, cudaStream_t s) {
  const int rounds = (int)std::max<int64_t>(1, ceil_div(count, CAP));
  for (int pass = 0; pass < 2; ++pass)
    for (int r = 0; r < rounds; ++r) {
      ClipTable<CAP> tab;
      std::memset(&tab, 0, sizeof(tab));
      tab.count = std::min(CAP, count - r * CAP);
      for (int k = 0; k < tab.count; ++k) {
        tab.data[k] = grads[r * CAP + k];
        tab.size[k] = sizes[r * CAP + k];
        tab.type[k] = (unsigned char)dtypes[r * CAP + k];
        tab.first[k + 1] = tab.first[k] + ceil_div(tab.size[k], kClipPiece);
      }
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr.val.programmaticStreamSerializationAllowed = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)ctas, 1, 1);
      cfg.blockDim = dim3(kClipThreads, 1, 1);
      cfg.stream = s;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (pass == 0)
        cudaLaunchKernelEx(&cfg, qlin_grad_norm_kernel<CAP>, tab, partials + (int64_t)r * ctas);
      else
        cudaLaunchKernelEx(&cfg, qlin_grad_scale_kernel<CAP>, tab, (const double*)partials, rounds * ctas, max_norm,
                           norm);
    }
}

// CTAs of the clipping kernels for a set of tensors: a batch of pieces each, at
// most what the device holds at once.
int clip_ctas(int64_t pieces, int sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(pieces, kClipBatch), (int64_t)kClipCtasPerSm * sms));
}

// Upper bound of the SM count, to size a workspace without a device.
constexpr int64_t kMostSms = 160;

}  // namespace

int qlin_mx_device_error(void* stream, int clear, int* device_status) {
  (void)stream;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, qlin::g_device_error, sizeof(int)) != cudaSuccess) return QLIN_ERR_LAUNCH;
  if (clear && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(qlin::g_device_error, &zero, sizeof(int)) != cudaSuccess) return QLIN_ERR_LAUNCH;
  }
  *device_status = v;
  return QLIN_OK;
}

extern "C" {

int qlin_mx_weights_size(int64_t K_g, int64_t N_g, size_t* bytes) {
  if (!bytes) return QLIN_ERR_ARG;
  const int st = check_groups(K_g, N_g);
  if (st == QLIN_OK) *bytes = (size_t)mx_bytes(K_g, N_g);
  return st;
}

int qlin_mx_quantize(int dtype, const void* wr, const void* wi, const void* wj, const void* wk, int64_t ld_w,
                     int64_t K_g, int64_t N_g, void* mx, void* stream) {
  int st = check_layer(dtype, 0, K_g, N_g, 0);
  if (st != QLIN_OK) return st;
  if (ld_w < K_g) return QLIN_ERR_SHAPE;
  if (!wr || !wi || !wj || !wk || !mx) return QLIN_ERR_ARG;
  if (!aligned(mx, 128)) return QLIN_ERR_ALIGN;
  int sms = 0;
  if ((st = qlin_host_device(&sms)) != QLIN_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaGetLastError();
  if (cudaMemsetAsync(mx, 0, kMxHeader, s) != cudaSuccess) return QLIN_ERR_LAUNCH;
  return by_type(dtype, [&](auto v) {
    using T = decltype(v);
    MxPlanes<const T> src;
    const void* w[4] = {wr, wi, wj, wk};
    bool vec = (ld_w * sizeof(T)) % 16 == 0;
    for (int c = 0; c < 4; ++c) {
      src.w[c] = static_cast<const T*>(w[c]);
      vec = vec && aligned(w[c], 16);
    }
    qlin_mx_quantize_kernel<T><<<record_grid(K_g, N_g, 3ll * sms), 256, 0, s>>>(src, ld_w, (int)K_g, (int)N_g,
                                                                         static_cast<uint8_t*>(mx), vec);
    return launched();
  });
}

int qlin_mx_dequantize(int dtype, const void* mx, int64_t K_g, int64_t N_g, void* wr, void* wi, void* wj, void* wk,
                       int64_t ld_w, void* stream) {
  int st = check_layer(dtype, 0, K_g, N_g, 0);
  if (st != QLIN_OK) return st;
  if (ld_w < K_g) return QLIN_ERR_SHAPE;
  if (!wr || !wi || !wj || !wk || !mx) return QLIN_ERR_ARG;
  if (!aligned(mx, 128)) return QLIN_ERR_ALIGN;
  int sms = 0;
  if ((st = qlin_host_device(&sms)) != QLIN_OK) return st;
  cudaGetLastError();
  return by_type(dtype, [&](auto v) {
    using T = decltype(v);
    const MxPlanes<T> dst = {{static_cast<T*>(wr), static_cast<T*>(wi), static_cast<T*>(wj), static_cast<T*>(wk)}};
    launch_dequantize<T>(mx, dst, ld_w, K_g, N_g, static_cast<cudaStream_t>(stream));
    return launched();
  });
}

int qlin_mx_workspace_size(int dtype, int64_t M, int64_t K_g, int64_t N_g, int rank, size_t* bytes) {
  if (!bytes) return QLIN_ERR_ARG;
  const int st = check_layer(dtype, M, K_g, N_g, rank);
  if (st == QLIN_OK) *bytes = M == 0 ? 0 : forward_ws(dtype, M, K_g, N_g, rank).total;
  return st;
}

int qlin_mx_forward(int dtype, const void* x, int64_t ld_x, const void* mx, const void* bias, const void* lora_a,
                    const void* lora_b, int rank, float lora_scale, void* y, int64_t ld_y, int64_t M, int64_t K_g,
                    int64_t N_g, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_layer(dtype, M, K_g, N_g, rank);
  if (st != QLIN_OK) return st;
  if (ld_x < 4 * K_g || ld_y < 4 * N_g) return QLIN_ERR_SHAPE;
  if (M == 0) return QLIN_OK;
  if (!x || !mx || !y || (rank > 0 && (!lora_a || !lora_b))) return QLIN_ERR_ARG;
  if (!aligned(mx, 128)) return QLIN_ERR_ALIGN;
  const ForwardWs w = forward_ws(dtype, M, K_g, N_g, rank);
  if (w.total > 0 && (!workspace || workspace_bytes < w.total || !aligned(workspace, 256))) return QLIN_ERR_WORKSPACE;
  int sms = 0;
  if ((st = qlin_host_device(&sms)) != QLIN_OK) return st;
  cudaGetLastError();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return by_type(dtype, [&](auto v) {
    using T = decltype(v);
    if (streams(dtype, M, N_g))
      return run_few<T>(dtype, static_cast<const T*>(x), ld_x, mx, static_cast<const T*>(bias),
                        static_cast<const T*>(lora_a), static_cast<const T*>(lora_b), rank, lora_scale,
                        static_cast<T*>(y), ld_y, M, K_g, N_g, ws, w, sms, static_cast<cudaStream_t>(stream));
    if constexpr (sizeof(T) == 2)
      return run_prefill<T>(static_cast<const T*>(x), ld_x, mx, static_cast<const T*>(bias),
                            static_cast<const T*>(lora_a), static_cast<const T*>(lora_b), rank, lora_scale,
                            static_cast<T*>(y), ld_y, M, K_g, N_g, ws, w, static_cast<cudaStream_t>(stream));
    return (int)QLIN_ERR_DTYPE;  // (fp32 always streams)
  });
}

int qlin_mx_backward_workspace_size(int dtype, int64_t M, int64_t K_g, int64_t N_g, int rank, size_t* bytes) {
  if (!bytes) return QLIN_ERR_ARG;
  const int st = check_layer(dtype, M, K_g, N_g, rank);
  if (st == QLIN_OK) *bytes = M == 0 ? 0 : backward_ws(dtype, M, K_g, N_g, rank).total;
  return st;
}

int qlin_mx_backward(int dtype, const void* gy, int64_t ld_g, const void* x, int64_t ld_x, const void* mx,
                     const void* lora_a, const void* lora_b, int rank, float lora_scale, void* dx, int64_t ld_dx,
                     void* da, void* db, void* dbias, int64_t M, int64_t K_g, int64_t N_g, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int st = check_layer(dtype, M, K_g, N_g, rank);
  if (st != QLIN_OK) return st;
  if (ld_g < 4 * N_g || (dx && ld_dx < 4 * K_g) || ((da || db) && ld_x < 4 * K_g)) return QLIN_ERR_SHAPE;
  if ((da || db) && rank == 0) return QLIN_ERR_ARG;
  if (M > 0 && (!gy || (dx && !mx) || ((da || db) && !x) || (rank > 0 && (!lora_a || !lora_b)))) return QLIN_ERR_ARG;
  if (!aligned(mx, 128)) return QLIN_ERR_ALIGN;
  const int64_t K = 4 * K_g, N = 4 * N_g;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M == 0) {  // empty sums
    if (!da && !db && !dbias) return QLIN_OK;
    cudaGetLastError();
    if (da) cudaMemsetAsync(da, 0, rank * K * elem(dtype), s);
    if (db) cudaMemsetAsync(db, 0, rank * N * elem(dtype), s);
    if (dbias) cudaMemsetAsync(dbias, 0, N * elem(dtype), s);
    return launched();
  }
  const BackwardWs w = backward_ws(dtype, M, K_g, N_g, rank);
  if (w.total > 0 && (!workspace || workspace_bytes < w.total || !aligned(workspace, 256))) return QLIN_ERR_WORKSPACE;
  int sms = 0;
  if ((st = qlin_host_device(&sms)) != QLIN_OK) return st;
  cudaGetLastError();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return by_type(dtype, [&](auto v) {
    using T = decltype(v);
    const T* g = static_cast<const T*>(gy);
    const T* xt = static_cast<const T*>(x);
    const T* a = static_cast<const T*>(lora_a);
    const T* b = static_cast<const T*>(lora_b);
    if constexpr (sizeof(T) == 2)
      return run_backward<T>(g, ld_g, xt, ld_x, mx, a, b, rank, lora_scale, static_cast<T*>(dx), ld_dx,
                             static_cast<T*>(da), static_cast<T*>(db), static_cast<T*>(dbias), M, K_g, N_g, ws, w, s);
    else
      return run_backward32(g, ld_g, xt, ld_x, mx, a, b, rank, lora_scale, static_cast<T*>(dx), ld_dx,
                            static_cast<T*>(da), static_cast<T*>(db), static_cast<T*>(dbias), M, K_g, N_g, ws, w, sms,
                            s);
  });
}

int qlin_grad_clip_workspace_size(int count, size_t* bytes) {
  if (!bytes) return QLIN_ERR_ARG;
  if (count < 0) return QLIN_ERR_SHAPE;
  *bytes = (size_t)(std::max<int64_t>(1, ceil_div(count, kClipTensors)) * kClipCtasPerSm * kMostSms * 8);
  return QLIN_OK;
}

int qlin_grad_clip(int count, void* const* grads, const int64_t* sizes, const int* dtypes, float max_norm,
                   float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0) return QLIN_ERR_SHAPE;
  if (!norm || (count > 0 && (!grads || !sizes || !dtypes)) || !(max_norm >= 0.f)) return QLIN_ERR_ARG;
  int64_t pieces = 0;
  for (int k = 0; k < count; ++k) {
    if (sizes[k] < 0) return QLIN_ERR_SHAPE;
    if (!known(dtypes[k])) return QLIN_ERR_DTYPE;
    if (sizes[k] > 0 && !grads[k]) return QLIN_ERR_ARG;
    if (!aligned(grads[k], (uintptr_t)elem(dtypes[k]))) return QLIN_ERR_ALIGN;
    pieces += ceil_div(sizes[k], kClipPiece);
  }
  size_t need = 0;
  qlin_grad_clip_workspace_size(count, &need);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) return QLIN_ERR_WORKSPACE;
  int sms = 0;
  const int st = qlin_host_device(&sms);
  if (st != QLIN_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaGetLastError();
  const int ctas = clip_ctas(pieces, (int)std::min<int64_t>(sms, kMostSms));
  double* partials = static_cast<double*>(workspace);
  if (count <= kClipFewTensors)
    clip_tables<kClipFewTensors>(count, grads, sizes, dtypes, max_norm, norm, partials, ctas, s);
  else
    clip_tables<kClipTensors>(count, grads, sizes, dtypes, max_norm, norm, partials, ctas, s);
  return launched();
}

}  // extern "C"
