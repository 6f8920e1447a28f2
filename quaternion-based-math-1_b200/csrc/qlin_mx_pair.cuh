// Many tokens through a layer with 4-bit weights, and the input gradient: the
// persistent CTA-pair kernel of qlin_pair.cuh (2-SM tcgen05 UMMA, the weight
// operand expanded into tensor memory, x straight from TMA) with two changes.
//
// Weights from codes (MX): a stage's 32 output x 32 input quaternions come as two
// records of 1088 bytes by bulk copy.  A builder lane (output quaternion o,
// component a) reads all four components of eight input quaternions in one
// 16-byte piece, expands them (mx_expand), multiplies by scale and sign of
// s(a, a^q) in one packed multiplication and pairs the components up: the
// expansion costs the integer pipe about 450 cycles of the 1024 that the eight
// UMMAs of a stage take at 256 tokens, and a quarter of a 16-bit layer's bytes.
// Without MX the weights are 16-bit component planes: the adjoint of the codes,
// times 2^-c.
// One set of builder warps could not keep up with the UMMAs on codes (a 4096 layer
// at 2048 tokens: 66 us, 57 on planes); two sets take every other stage each and need
// about 1080 cycles a stage, the integer pipe's time for it, just behind the UMMAs'
// 1024.  Tiles of 128 tokens, whose UMMAs take 512, are bound by that.
//
// Bound by the tensor pipe at 256 tokens (84 % of all cycles): 4096 -> 11008 at 2048
// bf16 tokens 113 us in a burst (1630 TFLOP/s), 134 us sustained (1380, at the power
// limit); 5120 -> 27648 with an adapter of rank 32 365 and 424 us.
//
// Adapter: y += t B^T with t = s x A^T and B as sums of bf16 parts, for fp16 too: bf16
// has fp32's range, so that neither a large B nor a small or large t leaves it.  t =
// t0 + t1 + t2 exactly; B is one part (bf16) or two (fp16: 11 bits as 8 + 3):
//     bf16  t0 B + t1 B + t2 B        fp16  t0 b0 + t1 b0 + t2 b0 + t0 b1 + t1 b1
// (t2 b1 is below 2^-24 of t B).  A stage holds the terms of up to 40 ranks (fp16: 24),
// part by part, and takes as many UMMAs as they need.  UMMAs with bf16 operands add to
// an accumulator that f16 ones began.  The builders fetch their rows of B before they
// wait for the stage.
//
// The accumulator holds y 2^-c (MxScaling); B is built with the same factor, and
// the epilogue multiplies by 2^c before the bias and the one rounding.
#pragma once

#include "qlin_mx.cuh"
#include "qlin_mx_few.cuh"
#include "qlin_pair.cuh"

namespace qlin {

constexpr int kMxPairBuilders = 8;  // warps 2-9: two sets of four, every other stage each
constexpr int kMxPairEpilogue = 8;  // warps 10-17: two sets of four, half of the tokens each
constexpr int kMxPairThreads = 32 * (2 + kMxPairBuilders + kMxPairEpilogue);

template <int NTOK, bool MX>
struct MxPairStage {
  static constexpr int kHalf = NTOK / 2;
  static constexpr int kXAtomBytes = kHalf * 128;
  static constexpr int kXBytes = 2 * kXAtomBytes;
  static constexpr int kWBytes = MX ? (2 * kMxRecord + 1023) / 1024 * 1024 : 4 * kPairWTileBytes;  // (two records, in whole KB)
  static constexpr int kStageBytes = kXBytes + kWBytes;
  // At 256 tokens x, W and the expanded rows share a ring position and a barrier;
  // at 128 the UMMAs of a stage take half as long, and x and W are fetched up to
  // seven stages ahead to cover their latency.
  static constexpr int kStages = NTOK == 256 ? kPairAStages : (MX ? 8 : 7);
  static constexpr bool kSplit = kStages != kPairAStages;
  static constexpr int kDBufs = NTOK == 256 ? 1 : 2;
  static constexpr int kAColBase = kDBufs * NTOK;
  static constexpr int kEpiOffset = kStages * kStageBytes;
  static constexpr int kBarOffset = kEpiOffset + 4 * kPairEpiBufBytes;  // two buffers per epilogue set
  static_assert(kBarOffset + 512 + 1024 <= kPairSmemBytes, "shared memory");
  static_assert(kStageBytes % 1024 == 0, "swizzled x tiles start on 1 KB");
  static_assert(kAColBase + kPairAStages * kPairACols <= 512, "tensor memory");
};

// Two elements of a row of B times `down` (a power of two) as bf16, and (fp16) the rest.
template <typename T>
__device__ __forceinline__ void mx_adapter_parts(uint32_t w, float down, uint32_t& first, uint32_t& second) {
  const T* e = reinterpret_cast<const T*>(&w);
  const float v0 = to_f32(e[0]) * down, v1 = to_f32(e[1]) * down;
  first = pack2<__nv_bfloat16>(v0, v1);
  const float r0 = v0 - __uint_as_float(first << 16), r1 = v1 - __uint_as_float(first & 0xFFFF0000u);
  second = pack2<__nv_bfloat16>(isfinite(r0) ? r0 : 0.f, isfinite(r1) ? r1 : 0.f);
}

// 32 lanes x 32 bit, four consecutive columns per thread.
__device__ __forceinline__ void tmem_st4(uint32_t taddr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(taddr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}

struct MxPairParams {
  const uint8_t* mx;    // codes
  const void* bias;
  const void* lora_b;   // [4 N_g, rank] or null
  void* y;
  int64_t ld_y;
  int M, N_g, K_g, rank;
  int kb, w_tiles;      // blocks of a row; 16-row tiles of the codes
  int stages;           // weight stages of a tile
  int ld_parts;         // rank in whole 16-byte pieces
  int lora_stages;      // ceil(ld_parts / kMxPairRanks)
  int nb_tiles, tiles;
  int wide;             // 16-byte output pieces are aligned
};

// Orders what other kernels stored before this thread's copies by the TMA unit.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async;" ::: "memory"); }

// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

template <typename T, int NTOK, bool MX>
__global__ void __launch_bounds__(kMxPairThreads, 1)
qlin_mx_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_t,
                    const __grid_constant__ CUtensorMap map_wr, const __grid_constant__ CUtensorMap map_wi,
                    const __grid_constant__ CUtensorMap map_wj, const __grid_constant__ CUtensorMap map_wk,
                    const MxPairParams prm) {
  using Cfg = MxPairStage<NTOK, MX>;
  constexpr bool HALF = std::is_same<T, __half>::value;
  constexpr uint32_t kIdesc = make_idesc_f16(256, NTOK, HALF ? 0u : 1u, false);
  constexpr uint32_t kIdescAdapter = make_idesc_f16(256, NTOK, 1u, false);
  constexpr int kParts = kMxPairParts<T>, kRanks = kMxPairRanks<T>;
  constexpr int S = Cfg::kStages, SA = kPairAStages, NB = Cfg::kDBufs;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);  // [S] x and W of this CTA landed
  uint64_t* empty = full + S;     // [S] the UMMAs of the stage completed (both CTAs)
  uint64_t* afull = empty + S;    // [SA] even CTA: both CTAs' builders wrote the expanded rows
  uint64_t* aempty = afull + SA;  // [SA] (kSplit) the UMMAs reading them completed (both CTAs)
  uint64_t* dfull = aempty + SA;  // [NB]
  uint64_t* dempty = dfull + NB;  // [NB], even CTA: both CTAs' epilogues drained the accumulator
  uint64_t* drain = dempty + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* issued = const_cast<int*>(abort_flag) + 1;  // producer: ring stages issued

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();     // 0: issues the UMMAs
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int my_tiles = pair < prm.tiles ? (prm.tiles - 1 - pair) / pairs + 1 : 0;
  const int nk = prm.stages + prm.lora_stages;
  const int total = my_tiles * nk;  // ring items of this pair

  if (prm.lora_stages == 0) pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SA; ++s) {
      mbar_init(&afull[s], 8);
      mbar_init(&aempty[s], 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(&dfull[b], 1);
      mbar_init(&dempty[b], 2 * kMxPairEpilogue);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *issued = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_x);
    if (prm.lora_stages) tma_prefetch_desc(&map_t);
    if constexpr (!MX) {
      tma_prefetch_desc(&map_wr);
      tma_prefetch_desc(&map_wi);
      tma_prefetch_desc(&map_wj);
      tma_prefetch_desc(&map_wk);
    }
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers initialised, tensor memory allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Everything below reads what earlier kernels of the stream wrote, or writes
  // what they may read.  After the down projection, which let this kernel start
  // only when everything before it had ended, t alone is waited for, by the
  // thread that fetches it (every output depends on it).
  if (prm.lora_stages == 0) pdl_wait_prior();

  auto tile_coords = [&](int t, int& n0, int& m0) {
    const int nb = t % prm.nb_tiles, tb = t / prm.nb_tiles;
    n0 = nb * 256 + (int)cta * kPairRows;  // this CTA's first real output
    m0 = tb * NTOK;                        // the pair's first token
  };
  const MxScaling<HALF> sc(prm.mx, prm.rank);
  const int c = sc.c;  // the accumulator holds y 2^-c

  if (warp == 0) {
    // ---------------- copies of this CTA's x half-tile and weights ----------------
    if (lane == 0) {
      const CUtensorMap* wmap[4] = {&map_wr, &map_wi, &map_wj, &map_wk};
      int g = 0;
      for (int j = 0; j < my_tiles && !*abort_flag; ++j) {
        int n0, m0;
        tile_coords(pair + j * pairs, n0, m0);
        const int mrow = m0 + (int)cta * Cfg::kHalf;
        const int tile0 = n0 / (4 * kMxRows), have = max(0, min(2, prm.w_tiles - tile0));
        for (int k = 0; k < nk; ++k, ++g) {
          const int s = g % S, n = g / S;
          if (n > 0 && !mbar_wait(&empty[s], (n - 1) & 1)) {
            *abort_flag = 1;
            break;
          }
          uint8_t* dst = smem + s * Cfg::kStageBytes;
          if (k >= prm.stages) {
            const int at = kRanks * kParts * (k - prm.stages);  // of the terms (zero past their end)
            if (j == 0 && at == 0) {
              pdl_wait_prior();
              // a kernel that starts from here on finds the down projection's results
              pdl_launch_dependents();
              fence_proxy_async();
            }
            mbar_arrive_expect_tx(&full[s], Cfg::kXBytes);
            tma_load_2d(dst, &map_t, &full[s], at, mrow);
            tma_load_2d(dst + Cfg::kXAtomBytes, &map_t, &full[s], at + 64, mrow);
          } else {
            mbar_arrive_expect_tx(&full[s], Cfg::kXBytes + (MX ? have * kMxRecord : 4 * kPairWTileBytes));
            tma_load_2d(dst, &map_x, &full[s], k * kPairStageK, mrow);
            tma_load_2d(dst + Cfg::kXAtomBytes, &map_x, &full[s], k * kPairStageK + 64, mrow);
            if constexpr (MX) {
              for (int h = 0; h < have; ++h)
                bulk_load(dst + Cfg::kXBytes + h * kMxRecord,
                          prm.mx + kMxHeader + ((int64_t)(tile0 + h) * prm.kb + k) * kMxRecord, kMxRecord, &full[s]);
            } else {
#pragma unroll
              for (int p = 0; p < 4; ++p)
                tma_load_2d(dst + Cfg::kXBytes + p * kPairWTileBytes, wmap[p], &full[s], k * (kPairStageK / 4),
                            n0 / 4);
            }
          }
          *issued = g + 1;
        }
        if (*abort_flag) break;
      }
    }
  } else if (warp == 1) {
    if (cta == 0) {
      // ---------------- UMMA issuer (even CTA) ----------------
      // The whole warp walks the loop, so that everything but the issue itself is
      // uniform; one elected lane issues.
      bool ok = true;
      int g = 0;
      for (int j = 0; j < my_tiles && ok; ++j) {
        const int b = j % NB, u = j / NB;
        if (u > 0 && !mbar_wait(&dempty[b], (u - 1) & 1)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        for (int k = 0; k < nk && ok; ++k, ++g) {
          const int s = g % S, sa = g % SA;
          // both CTAs' builders arrive only after their own CTA's x and W of
          // this stage landed: this one wait covers the B operand too
          ok = __all_sync(0xffffffffu, mbar_wait(&afull[sa], (g / SA) & 1) && !*abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t bdesc0 = smem_desc_sw128(smem + s * Cfg::kStageBytes);
          const uint32_t d = tmem + b * NTOK, a0 = tmem + Cfg::kAColBase + sa * kPairACols;
          const bool adapter = k >= prm.stages;
          const uint32_t idesc = adapter ? kIdescAdapter : kIdesc;
          const int steps = adapter ? (kParts * min(kRanks, prm.ld_parts - kRanks * (k - prm.stages)) + 15) / 16
                                    : kPairStageK / 16;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kPairStageK / 16; ++kk)
              if (kk < steps)
                umma_pair_ts(d, a0 + 8 * kk, bdesc0 + (uint64_t)((kk >> 2) * (Cfg::kXAtomBytes >> 4)) + 2 * (kk & 3),
                             idesc, (k > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(&empty[s], 0x3);
            if constexpr (Cfg::kSplit) umma_commit_pair(&aempty[sa], 0x3);
            if (k == nk - 1) umma_commit_pair(&dfull[b], 0x3);
          }
          __syncwarp();
        }
      }
      if (elect_one()) {
        if (!ok) *abort_flag = 1;
        // every UMMA issued above has completed before the teardown
        umma_commit_pair(drain, 0x1);
        mbar_wait(drain, 0, 50000000ull);
      }
      __syncwarp();
    }
  } else if (warp < 2 + kMxPairBuilders) {
    // ---------------- builders: expanded weight rows into tensor memory ----------------
    // Lane l of builder warp w writes tensor-memory lane 32 q + l (q = w % 4):
    // output quaternion n0/4 + 8 q + l % 8, component a = l / 8.
    const int quarter = warp & 3;
    const int a = lane >> 3;
    const int row = 8 * quarter + (lane & 7);  // of the CTA's 32 output quaternions
    uint32_t sign[4];                          // of s(a, a^q), on both halves
#pragma unroll
    for (int q = 0; q < 4; ++q) sign[q] = (mx_negative(a) >> (a ^ q) & 1) ? 0x80008000u : 0u;
    const uint32_t tm_lane = (uint32_t)(32 * quarter) << 16;
    const MxPowers pw;
    const float down = scalbnf(1.f, -c);
    const int set = (warp - 2) >> 2;
    int k = set, j = 0;
    for (int g = set; g < total; g += 2, k += 2) {
      while (k >= nk) {
        k -= nk;
        ++j;
      }
      // (in a shared ring x and W are fetched once the position's UMMAs are done, so
      // its tensor memory is free too when they land)
      const int s = g % S, sa = g % SA;
      const int r0 = kRanks * (k - prm.stages);  // (an adapter's stage: its ranks)
      uint4 brow[kRanks / 8];
      if (k >= prm.stages) {
        int n0, m0;
        tile_coords(pair + j * pairs, n0, m0);
        const int64_t n_out = n0 + 4 * row + a;
        const T* b = reinterpret_cast<const T*>(prm.lora_b) + n_out * prm.rank + r0;
        const int left = n_out < 4 * (int64_t)prm.N_g ? prm.rank - r0 : 0;
        const bool vec = prm.rank % 8 == 0 && (reinterpret_cast<uintptr_t>(prm.lora_b) & 15) == 0;
#pragma unroll
        for (int e = 0; e < kRanks / 8; ++e) {
          brow[e] = make_uint4(0u, 0u, 0u, 0u);
          if (vec) {
            if (8 * e < left) brow[e] = ld_cg_v4(b + 8 * e);
          } else {
            unsigned short h[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
              h[u] = 8 * e + u < left ? *reinterpret_cast<const volatile unsigned short*>(b + 8 * e + u) : (unsigned short)0;
            brow[e] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                                 h[6] | (uint32_t)h[7] << 16);
          }
        }
      }
      bool ok = !*abort_flag && mbar_wait(&full[s], (g / S) & 1);
      if (Cfg::kSplit && ok && g >= SA) ok = mbar_wait(&aempty[sa], (g / SA - 1) & 1);
      if (!ok) *abort_flag = 1;
      const uint32_t col = tmem + tm_lane + Cfg::kAColBase + sa * kPairACols;
      if (!*abort_flag && k >= prm.stages) {
        const int ranks = min(kRanks, prm.ld_parts - r0);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < kRanks / 8; ++e) {
          if (8 * e >= ranks) break;
          uint32_t p0[4], p1[4];
          const uint32_t w[4] = {brow[e].x, brow[e].y, brow[e].z, brow[e].w};
#pragma unroll
          for (int u = 0; u < 4; ++u) mx_adapter_parts<T>(w[u], down, p0[u], p1[u]);
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const uint32_t at = col + (part * ranks + 8 * e) / 2;
            if (part < 3) tmem_st4(at, p0[0], p0[1], p0[2], p0[3]);
            else tmem_st4(at, p1[0], p1[1], p1[2], p1[3]);
          }
        }
        // (the last UMMA's second half where the terms end in its first)
        if (kParts * ranks % 16) tmem_st4(col + kParts * ranks / 2, 0u, 0u, 0u, 0u);
        tmem_st_wait();
      } else if (!*abort_flag && MX) {
        const uint32_t rec = smem_u32(smem + s * Cfg::kStageBytes + Cfg::kXBytes) + (quarter >> 1) * kMxRecord;
        const int r16 = row & 15;
        const uint32_t scales = lds32(rec + kMxCodeBytes + r16 * 4);
        uint32_t mult[4];  // of component a^q, with its sign
#pragma unroll
        for (int q = 0; q < 4; ++q) mult[q] = mx_multiplier<HALF>((scales >> (8 * (a ^ q))) & 255u, sc.off) ^ sign[q];
        auto expand = [&](auto far) {
          constexpr bool FAR = decltype(far)::value;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
#pragma unroll
            for (int o = 0; o < 2; ++o) {  // octet 2h + o: columns 16 of 32
              const uint4 w4 = lds128(rec + r16 * 64 + (2 * h + o) * 16);
              uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
              if (a & 1) {
                uint32_t x = w[0]; w[0] = w[1]; w[1] = x;
                x = w[2]; w[2] = w[3]; w[3] = x;
              }
              if (a & 2) {
                uint32_t x = w[0]; w[0] = w[2]; w[2] = x;
                x = w[1]; w[1] = w[3]; w[3] = x;
              }
              uint32_t e[4][4];
#pragma unroll
              for (int q = 0; q < 4; ++q) mx_expand_scaled<HALF, FAR>(pw, w[q], mult[q], e[q]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                r[16 * o + 2 * i] = __byte_perm(e[0][i], e[1][i], 0x5410);
                r[16 * o + 2 * i + 1] = __byte_perm(e[2][i], e[3][i], 0x5410);
                r[16 * o + 8 + 2 * i] = __byte_perm(e[0][i], e[1][i], 0x7632);
                r[16 * o + 8 + 2 * i + 1] = __byte_perm(e[2][i], e[3][i], 0x7632);
              }
            }
            __syncwarp();
            tmem_st32(col + 32 * h, r);
          }
        };
        if (HALF && sc.far) expand(std::integral_constant<bool, HALF>());
        else expand(std::false_type());
        tmem_st_wait();
      } else if (!*abort_flag) {
        // W_a[o, 32 inputs]: 64 bytes, chunk u at chunk u ^ ((row >> 1) & 3) (64-byte swizzle);
        // W_{a^q'} from lanes l ^ 8 q' (same o)
        const uint32_t wrow =
            smem_u32(smem + s * Cfg::kStageBytes + Cfg::kXBytes + a * kPairWTileBytes + row * 64);
        uint32_t w0[16];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint4 v = lds128(wrow + ((u ^ ((row >> 1) & 3)) << 4));
          w0[4 * u] = v.x; w0[4 * u + 1] = v.y; w0[4 * u + 2] = v.z; w0[4 * u + 3] = v.w;
        }
        const uint32_t sg01 = (sign[0] & 0x8000u) | (sign[1] & 0x80000000u);
        const uint32_t sg23 = (sign[2] & 0x8000u) | (sign[3] & 0x80000000u);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
#pragma unroll
          for (int e8 = 0; e8 < 8; ++e8) {
            const uint32_t v0 = w0[8 * h + e8];
            const uint32_t v1 = __shfl_xor_sync(0xffffffffu, v0, 8);
            const uint32_t v2 = __shfl_xor_sync(0xffffffffu, v0, 16);
            const uint32_t v3 = __shfl_xor_sync(0xffffffffu, v0, 24);
            r[4 * e8 + 0] = __byte_perm(v0, v1, 0x5410) ^ sg01;
            r[4 * e8 + 1] = __byte_perm(v2, v3, 0x5410) ^ sg23;
            r[4 * e8 + 2] = __byte_perm(v0, v1, 0x7632) ^ sg01;
            r[4 * e8 + 3] = __byte_perm(v2, v3, 0x7632) ^ sg23;
          }
          tmem_st32(col + 32 * h, r);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&afull[sa], 0);
    }
  } else {
    // ---------------- epilogue ----------------
    // Drain the accumulator into registers (scaled, bias added, rounded, two
    // tokens per word), release it to the UMMA issuer, then store through a
    // shared-memory transpose.
    const int quarter = warp & 3;
    const int half = (warp - 2 - kMxPairBuilders) >> 2;  // of the tile's tokens
    const int et = (threadIdx.x - 32 * (2 + kMxPairBuilders)) & 127;
    constexpr int kTok = NTOK / 2;
    const int n_local = 32 * quarter + 4 * (lane & 7) + (lane >> 3);
    const float factor = scalbnf(1.f, c);
    T* y = reinterpret_cast<T*>(prm.y);
    const T* bias = reinterpret_cast<const T*>(prm.bias);
    for (int j = 0; j < my_tiles; ++j) {
      const int b = j % NB, u = j / NB;
      int n0, m0;
      tile_coords(pair + j * pairs, n0, m0);
      const bool got = !*abort_flag && mbar_wait(&dfull[b], u & 1);
      if (!got) *abort_flag = 1;
      tc_fence_after();
      const int n = n0 + n_local;
      const float bv = (bias && n < 4 * prm.N_g) ? to_f32(bias[n]) : 0.f;
      uint32_t packed[kTok / 2];
#pragma unroll
      for (int q = 0; q < kTok / 32; ++q) {
        uint32_t v[32];
        if (got) {
          __syncwarp();
          tmem_ld32(tmem + ((uint32_t)(32 * quarter) << 16) + b * NTOK + half * kTok + 32 * q, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int t = 0; t < 32; ++t) v[t] = 0u;
        }
#pragma unroll
        for (int t = 0; t < 16; ++t)
          packed[16 * q + t] = pack2<T>(fmaf(__uint_as_float(v[2 * t]), factor, bv),
                                        fmaf(__uint_as_float(v[2 * t + 1]), factor, bv));
      }
      // this warp has read its lanes of the accumulator: the even CTA may reuse it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&dempty[b], 0);
#pragma unroll
      for (int grp = 0; grp < kTok / kPairEpiTokens; ++grp) {
        T* stage = reinterpret_cast<T*>(smem + Cfg::kEpiOffset + (2 * half + (grp & 1)) * kPairEpiBufBytes);
        unsigned short* st16 = reinterpret_cast<unsigned short*>(stage);
#pragma unroll
        for (int t2 = 0; t2 < kPairEpiTokens / 2; ++t2) {
          const uint32_t wv = packed[(kPairEpiTokens / 2) * grp + t2];
          st16[(2 * t2) * kPairRows + n_local] = (unsigned short)(wv & 0xffffu);
          st16[(2 * t2 + 1) * kPairRows + n_local] = (unsigned short)(wv >> 16);
        }
        asm volatile("bar.sync %0, %1;" ::"r"(kPairEpiBar + half), "n"(128) : "memory");
        if (got) {
          // 16 tokens x 128 outputs = 256 pieces of 16 bytes, two per thread
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = et + 128 * h, t = at >> 4, cc = at & 15;
            const int m = m0 + half * kTok + kPairEpiTokens * grp + t, nn = n0 + 8 * cc;
            if (m < prm.M && nn < 4 * prm.N_g) {
              const uint4 v = *reinterpret_cast<const uint4*>(stage + t * kPairRows + 8 * cc);
              T* out = y + (int64_t)m * prm.ld_y + nn;
              if (prm.wide) {
                *reinterpret_cast<uint4*>(out) = v;
              } else {  // an odd number of output quaternions: 8-byte pieces
                *reinterpret_cast<uint2*>(out) = make_uint2(v.x, v.y);
                if (nn + 4 < 4 * prm.N_g) *reinterpret_cast<uint2*>(out + 4) = make_uint2(v.z, v.w);
              }
            }
          }
        }
      }
    }
  }

  // ---------------- teardown ----------------
  __syncwarp();
  if (threadIdx.x == 0 && *abort_flag) {
    // let issued copies land before the shared memory goes away
    const int g1 = *issued;
    for (int g = g1 - S > 0 ? g1 - S : 0; g < g1; ++g) mbar_wait(&full[g % S], (g / S) & 1, 50000000ull);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while the other may still use its memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace qlin
