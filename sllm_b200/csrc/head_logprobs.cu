// Log-probabilities and entropies of the logits  z[m, n] = sum_k X[m, k] W[n, k]  (bf16 operands; with a soft cap c: c tanh(z / c))
// that never leave the chip: a tile of logits becomes three numbers per row,
//   m = max z,  S = sum 2^((z - m) log2 e),  W = sum 2^t t of the same t = (z - m) log2 e,
// and a second kernel joins a row's parts.  The row's given token leaves its logit behind on the way.
//
// What bounds it: few rows the reading of W, many rows the tensor cores (2 m n k operations).  Persistent CTA pairs (cta_group::2) on
// tiles of 256 rows x BN tokens, as in gemm_prompt.cu:
//   warp 0      producer: each CTA copies its 128 rows of X and BN / 2 rows of W per 128-byte K block; the bytes of both CTAs
//               count on the first CTA's barrier
//   warp 1      owns the tensor memory; in the first CTA it issues the products for both
//   warps 4 ..  two groups of four, thread = row, a group per half of the tile's columns
// Measured (B200, one launch and the join, m x n x k, us, in brackets what the rates of a copy and of a library product give; calls a
// few at a time, and behind the stroke one after another for seconds, where the power limit holds the clock at 1.1 to 1.3 GHz):
//      1 x 128256 x 4096     171 / 184 (163)         777 x 151936 x 2560, cap    536 / 628 (361: 777 rows fill 3.04 tiles)
//     48 x 201088 x 2880     186 / 206 (179)        4096 x 128256 x 4096        2784 / 3117 (2571; 3119 at the sustained rate)
// The tensor pipe is busy for 0.89 of the third's cycles (0.98 without the cap), the DRAM at 0.78 of its peak in the first two.
// The first two through the kernel for few rows; on CTA pairs, whose second half has no rows there, they took 270 and 260.
// A tile's sum over K is taken in chains of kHlChain K blocks with an accumulator of their own, which the epilogue warps add in fp32
// registers while the next chain is multiplied: tensor memory rounds towards zero, and a chain's error grows with its length (4096 wide:
// 2.3e-7 of the log-probabilities with chains of 8, 4.6e-7 with 16, 9.7e-7 with 32, which takes 1 % less time).
#include <atomic>
#include "pair_mma.cuh"
#include "api.h"
#include "tmap.h"

namespace sllm {

constexpr int kHlRows = 128;                // rows of X per CTA
constexpr int kHlMaxStages = 9;
constexpr int kHlGroupN = 8;                // columns of tiles per raster group
constexpr int kHlChain = 8;                 // K blocks of 64 added in tensor memory
constexpr int kHlThreads = 384;

template <int BN>
struct HlShape {
  static constexpr int kABytes = kHlRows * 128;
  static constexpr int kBBytes = BN / 2 * 128;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 7 : 9;
  static constexpr int kCols = BN / 2;      // columns per epilogue thread
  static constexpr int kAcc = 512 / BN;
  static constexpr uint32_t kTmem = 512;
};

struct __align__(16) HlShared {
  uint64_t full[kHlMaxStages];              // first CTA's: the bytes of both
  uint64_t empty[kHlMaxStages];
  uint64_t acc_full[4];
  uint64_t acc_empty[4];                    // first CTA's: the epilogue warps of both
  uint32_t tmem_base;
  int abort_flag;
};

struct HlParams {
  int m, n, num_kb, chains, tiles_m, tiles_n;
  float cap, inv_cap;                       // 0: none
  const int* tokens;                        // [m]
  float4* part;                             // [2 tiles_n, m]: m, S, W
  float* given;                             // [m]: the token's logit
  int* status;
};

constexpr float kHlLog2e = 1.4426950408889634f, kHlLn2 = 0.6931471805599453f;

__device__ __forceinline__ void hl_tile(const HlParams& p, int t, int& tm, int& tn) {
  const int per = kHlGroupN * p.tiles_m, g = t / per, r = t - g * per, wide = min(kHlGroupN, p.tiles_n - g * kHlGroupN);
  tm = r / wide;
  tn = g * kHlGroupN + r - tm * wide;
}
__device__ __forceinline__ float hl_exp2(float x) {            // 0 below the smallest normal number
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float hl_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sums of some logits of a row.
struct HlSums {
  float m, s, w;
  __device__ __forceinline__ void add(float om, float os, float ow) {      // NaN passes through
    const float top = fmaxf(m, om);
    const float t = m == top ? 0.f : fmaxf((m - top) * kHlLog2e, -1000.f), e = hl_exp2(t);
    const float u = om == top ? 0.f : fmaxf((om - top) * kHlLog2e, -1000.f), f = hl_exp2(u);
    w = e * fmaf(t, s, w) + f * fmaf(u, os, ow);
    s = e * s + f * os;
    m = top;
  }
};

// z <- cap tanh(z / cap).  Logits are small beside the cap as a rule: tanh(u) = u + u^3 P(u^2) below kHlSmall, P of degree 4 fitted to the least
// relative error there (3e-9; 7e-8 with its roundings), and 1 - 2 / (1 + e^2u) beyond (1.6e-7).  With tanhf a tile of 128 columns took 9000
// cycles of its thread in place of 3500.
constexpr float kHlSmall = 0.6f;
template <int kCols>
__device__ __forceinline__ void hl_cap(const HlParams& p, float (&z)[kCols]) {
  const uint64_t inv = pack_f32x2(p.inv_cap, p.inv_cap), cap = pack_f32x2(p.cap, p.cap);
  auto both = [](float x) { return pack_f32x2(x, x); };
  const float bound = kHlSmall * p.cap;
#pragma unroll
  for (int c0 = 0; c0 < kCols; c0 += 8) {
    float top = 0.f;
#pragma unroll
    for (int c = c0; c < c0 + 8; ++c) top = fmaxf(top, fabsf(z[c]));
    if (top < bound) {
#pragma unroll
      for (int c = c0; c < c0 + 8; c += 2) {
        const uint64_t u = mul_f32x2(pack_f32x2(z[c], z[c + 1]), inv), s = mul_f32x2(u, u);
        uint64_t q = fma_f32x2(both(-0.005895140671612253f), s, both(0.020795955859865982f));
        q = fma_f32x2(q, s, both(-0.05378382526597832f));
        q = fma_f32x2(q, s, both(0.1333192406261711f));
        q = fma_f32x2(q, s, both(-0.3333329799945037f));
        const float2 y = unpack_f32x2(mul_f32x2(fma_f32x2(u, mul_f32x2(q, s), u), cap));
        z[c] = y.x;
        z[c + 1] = y.y;
      }
    } else {
#pragma unroll
      for (int c = c0; c < c0 + 8; ++c) {
        const float u = z[c] * p.inv_cap, a = fabsf(u), s = u * u;
        const float q = fmaf(fmaf(fmaf(fmaf(-0.005895140671612253f, s, 0.020795955859865982f), s, -0.05378382526597832f), s, 0.1333192406261711f), s,
                             -0.3333329799945037f);
        const float far = 1.f - __fdividef(2.f, 1.f + hl_exp2(2.f * kHlLog2e * a));
        z[c] = p.cap * (a < kHlSmall ? fmaf(u, q * s, u) : copysignf(far, u));      // (NaN: far, a NaN)
      }
    }
  }
}

// The part of a row that lies in columns n0 .. n0 + width - 1 (nothing with width <= 0): caps the logits, leaves the given token's behind and
// sums up.  All lanes of a warp take part.
template <int kCols>
__device__ __forceinline__ HlSums hl_reduce(const HlParams& p, float (&z)[kCols], int token, int row, int n0, int width) {
  if (p.cap > 0.f) hl_cap<kCols>(p, z);
  const int at = token - n0;
  const bool here = token >= n0 && at < width;
  if (__any_sync(0xffffffffu, here)) {
    float x = 0.f;
#pragma unroll
    for (int c = 0; c < kCols; ++c) x = at == c ? z[c] : x;
    if (here) p.given[row] = x;
  }
  if (width < kCols) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) z[c] = c < width ? z[c] : -INFINITY;
  }
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < kCols; c += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) m4[i] = fmaxf(m4[i], z[c + i]);
  const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
  float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
  if (m < INFINITY) {
    const float ref = m > -INFINITY ? m : 0.f;             // (nothing but -inf: every term is 2^-1000)
    const uint64_t minus = pack_f32x2(-ref, -ref), log2e = pack_f32x2(kHlLog2e, kHlLog2e);
    uint64_t s = 0ull, w = 0ull;
#pragma unroll
    for (int c = 0; c < kCols; c += 2) {
      const float2 d = unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(z[c], z[c + 1]), minus), log2e));
      const float t0 = hl_max_nan(d.x, -1000.f), t1 = hl_max_nan(d.y, -1000.f);
      const uint64_t e = pack_f32x2(hl_exp2(t0), hl_exp2(t1));
      s = add_f32x2(s, e);
      w = fma_f32x2(e, pack_f32x2(t0, t1), w);
    }
    const float2 s2 = unpack_f32x2(s), w2 = unpack_f32x2(w);
    s0 = s2.x;
    s1 = s2.y;
    w0 = w2.x;
    w1 = w2.y;
  } else {                                                 // uniform over +inf
#pragma unroll
    for (int c = 0; c < kCols; ++c) s0 += z[c] != z[c] ? z[c] : z[c] == INFINITY ? 1.f : 0.f;
  }
  return {m, s0 + s1, w0 + w1};
}

template <int BN>
__global__ void __launch_bounds__(kHlThreads, 1)
head_logprobs_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const HlParams p) {
  using S = HlShape<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  HlShared* sh = reinterpret_cast<HlShared*>(smem + S::kStages * S::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank()), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.tiles_m * p.tiles_n;
  volatile int* abort_flag = &sh->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
    }
    for (int b = 0; b < S::kAcc; ++b) {
      mbar_init(&sh->acc_full[b], 1);
      mbar_init(&sh->acc_empty[b], 2 * 8);
    }
    sh->abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) pair_tmem_alloc(&sh->tmem_base, S::kTmem);
  tc_fence_before();
  __syncthreads();
  cluster_sync_pair();                                     // both CTAs' barriers exist and both hold their tensor memory
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;

  if (warp < 4) {
    // 128 x 72 + 256 x 216 of the 384 x 168 registers of the launch
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      if (elect_one()) {
        pdl_wait();
        int it = 0;                                        // K blocks over all tiles
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += pairs) {
          int tm, tn;
          hl_tile(p, t, tm, tn);
          for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
            const int s = it % S::kStages;
            if (it >= S::kStages &&
                !mbar_wait(&sh->empty[s], ((it / S::kStages) & 1) ^ 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_SMEM_EMPTY)) {
              ok = false;
              break;
            }
            if (rank == 0) mbar_expect_tx(&sh->full[s], 2 * S::kStage);
            const uint32_t full = leader_addr(&sh->full[s]);
            pair_tma_load_2d(smem + s * S::kStage + S::kABytes, &tm_w, full, kb * 64, tn * BN + rank * (BN / 2));
            pair_tma_load_2d(smem + s * S::kStage, &tm_x, full, kb * 64, (tm * 2 + rank) * kHlRows);
          }
        }
        pdl_trigger();
        // every copy has landed before the pair may leave (at once unless something gave up): a stage's last fill
        if (rank == 0) {
          int dummy = 0;
          for (int j = max(0, it - S::kStages); j < it; ++j)
            mbar_wait(&sh->full[j % S::kStages], (j / S::kStages) & 1, &dummy, p.status, SLLM_DEV_TIMEOUT_DRAIN, 200000000LL);
        }
      }
      __syncwarp();
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t idesc = make_idesc(kFmtBf16, 256, BN);
      int it = 0, acc = 0;                                 // acc: accumulators handed over so far
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
          const int s = it % S::kStages, buf = acc % S::kAcc;
          const bool first = kb % kHlChain == 0, last = kb % kHlChain == kHlChain - 1 || kb == p.num_kb - 1;
          ok = mbar_wait(&sh->full[s], (it / S::kStages) & 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_TMA_FULL);
          if (ok && first) ok = mbar_wait(&sh->acc_empty[buf], ((acc / S::kAcc) & 1) ^ 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_TMEM_EMPTY);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * S::kStage);
          const uint64_t ad = make_smem_desc_sw128(a_addr), bd = make_smem_desc_sw128(a_addr + S::kABytes);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)                    // 4 x 32 bytes of K
              pair_umma<false>(tmem_base + buf * BN, ad + 2 * k, bd + 2 * k, idesc, k > 0 || !first);
            pair_commit(&sh->empty[s]);
            if (last) pair_commit(&sh->acc_full[buf]);
          }
          __syncwarp();
          acc += last;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    pdl_wait();
    const int q = warp & 3, grp = (warp - 4) >> 2;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + grp * S::kCols;
    const uint32_t empty_addr = leader_addr(&sh->acc_empty[0]);
    int acc = 0;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      int tm, tn;
      hl_tile(p, t, tm, tn);
      const int row = (tm * 2 + rank) * kHlRows + q * 32 + lane, n0 = tn * BN + grp * S::kCols;
      const int token = row < p.m ? p.tokens[row] : -1;
      float z[S::kCols];
#pragma unroll
      for (int c = 0; c < S::kCols; ++c) z[c] = 0.f;
      for (int chain = 0; chain < p.chains; ++chain, ++acc) {
        ok = mbar_wait(&sh->acc_full[acc % S::kAcc], (acc / S::kAcc) & 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_TMEM_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < S::kCols / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(lane_addr + (acc % S::kAcc) * BN + c * 32, r);
          tmem_wait_regs(r);
#pragma unroll
          for (int j = 0; j < 32; ++j) z[c * 32 + j] += __uint_as_float(r[j]);
        }
        tc_fence_before();                                 // all of it is in registers
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(empty_addr + 8 * (acc % S::kAcc));
      }
      if (!ok) break;
      const HlSums part = hl_reduce<S::kCols>(p, z, token, row, n0, min(p.n - n0, S::kCols));
      if (row < p.m) p.part[static_cast<size_t>(2 * tn + grp) * p.m + row] = make_float4(part.m, part.s, part.w, 0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_pair();                                     // nothing of the other CTA reaches this one any more
  if (warp == 1) {
    tc_fence_after();
    pair_tmem_dealloc(tmem_base, S::kTmem);
  }
}

// Up to 128 rows, where the reading of W is what there is to do: one CTA per SM with an equal share of W's rows (kHfBox of them to
// a copy), so that no CTA reads longer than the others, in tiles of up to 256.  One tensor-core row is one row of X; a CTA's tiles
// belong to the same rows, whose sums stay in registers until the end.  CTAs begin at different K blocks: all of them reading the same line
// of a single row of X at a time cost 7 % (1 x 128256 x 4096: 218 us, 204 with turns), and copies of 128 rows for one 8 % more (187 with 8).
constexpr int kHfBox = 16, kHfTile = 256, kHfStages = 4, kHfCols = kHfTile / 2;
constexpr int kHfABytes = kHlRows * 128, kHfStage = kHfABytes + kHfTile * 128;

__global__ void __launch_bounds__(kHlThreads, 1)
head_few_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const HlParams p, int share, int x_rows) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  HlShared* sh = reinterpret_cast<HlShared*>(smem + kHfStages * kHfStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first_n = blockIdx.x * share, last_n = min(first_n + share, p.n);      // the CTA's columns
  volatile int* abort_flag = &sh->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kHfStages; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh->acc_full[b], 1);
      mbar_init(&sh->acc_empty[b], 8);
    }
    sh->abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) {
    tmem_alloc(&sh->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      if (elect_one()) {
        pdl_wait();
        const int turn = static_cast<int>(blockIdx.x * static_cast<long long>(p.num_kb) / gridDim.x);
        int it = 0;                                        // K blocks over all tiles
        bool ok = true;
        for (int n0 = first_n; ok && n0 < last_n; n0 += kHfTile) {
          const int boxes = (min(kHfTile, last_n - n0) + kHfBox - 1) / kHfBox;
          for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
            const int s = it % kHfStages;
            if (it >= kHfStages && !mbar_wait(&sh->empty[s], ((it / kHfStages) & 1) ^ 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_SMEM_EMPTY)) {
              ok = false;
              break;
            }
            uint8_t* dst = smem + s * kHfStage;
            mbar_expect_tx(&sh->full[s], x_rows * 128 + boxes * kHfBox * 128);
            int k0 = kb + turn;
            k0 = (k0 < p.num_kb ? k0 : k0 - p.num_kb) * 64;
            for (int b = 0; b < boxes; ++b) tma_load_2d(dst + kHfABytes + b * kHfBox * 128, &tm_w, &sh->full[s], k0, n0 + b * kHfBox);
            tma_load_2d(dst, &tm_x, &sh->full[s], k0, 0);
          }
        }
        pdl_trigger();
        // every copy has landed before the CTA may leave (at once unless something gave up): a stage's last fill
        int dummy = 0;
        for (int j = max(0, it - kHfStages); j < it; ++j)
          mbar_wait(&sh->full[j % kHfStages], (j / kHfStages) & 1, &dummy, p.status, SLLM_DEV_TIMEOUT_DRAIN, 200000000LL);
      }
      __syncwarp();
    } else if (warp == 1) {
      int it = 0, acc = 0;                                 // acc: accumulators handed over so far
      bool ok = true;
      for (int n0 = first_n; ok && n0 < last_n; n0 += kHfTile) {
        const int boxes = (min(kHfTile, last_n - n0) + kHfBox - 1) / kHfBox;
        const uint32_t idesc = make_idesc(kFmtBf16, 128, boxes * kHfBox);
        for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
          const int s = it % kHfStages, buf = acc & 1;
          const bool first = kb % kHlChain == 0, last = kb % kHlChain == kHlChain - 1 || kb == p.num_kb - 1;
          ok = mbar_wait(&sh->full[s], (it / kHfStages) & 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_TMA_FULL);
          if (ok && first) ok = mbar_wait(&sh->acc_empty[buf], ((acc / 2) & 1) ^ 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_TMEM_EMPTY);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * kHfStage);
          const uint64_t ad = make_smem_desc_sw128(a_addr), bd = make_smem_desc_sw128(a_addr + kHfABytes);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16(tmem_base + buf * kHfTile, ad + 2 * k, bd + 2 * k, idesc, k > 0 || !first);
            tc_commit(&sh->empty[s]);
            if (last) tc_commit(&sh->acc_full[buf]);
          }
          __syncwarp();
          acc += last;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    pdl_wait();
    const int q = warp & 3, grp = (warp - 4) >> 2, row = q * 32 + lane;
    const bool idle = q * 32 >= p.m;                       // a warp without rows only hands the accumulators back
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + grp * kHfCols;
    const int token = row < p.m ? p.tokens[row] : -1;
    HlSums all = {-INFINITY, 0.f, 0.f};
    int acc = 0;
    bool ok = true;
    for (int n0 = first_n; ok && n0 < last_n; n0 += kHfTile) {
      const int mine = n0 + grp * kHfCols, width = min(last_n - mine, kHfCols);
      const bool skip = idle || width <= 0;
      float z[kHfCols];
#pragma unroll
      for (int c = 0; c < kHfCols; ++c) z[c] = 0.f;
      for (int chain = 0; chain < p.chains; ++chain, ++acc) {
        ok = mbar_wait(&sh->acc_full[acc & 1], (acc / 2) & 1, abort_flag, p.status, SLLM_DEV_TIMEOUT_TMEM_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (!skip) {
#pragma unroll
          for (int c = 0; c < kHfCols / 32; ++c) {
            if (c * 32 >= width) break;                    // (columns of no product are not read)
            uint32_t r[32];
            tmem_ld32(lane_addr + (acc & 1) * kHfTile + c * 32, r);
            tmem_wait_regs(r);
#pragma unroll
            for (int j = 0; j < 32; ++j) z[c * 32 + j] += __uint_as_float(r[j]);
          }
        }
        tc_fence_before();                                 // all of it is in registers
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->acc_empty[acc & 1]);
      }
      if (!ok) break;
      if (!skip) {
        const HlSums part = hl_reduce<kHfCols>(p, z, token, row, mine, width);
        all.add(part.m, part.s, part.w);
      }
    }
    if (row < p.m) p.part[static_cast<size_t>(2 * blockIdx.x + grp) * p.m + row] = make_float4(all.m, all.s, all.w, 0.f);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// The parts of a row: eight rows per CTA, so that a line of parts is read as a whole, 128 threads for each.
constexpr int kHlJoinRows = 8, kHlJoinThreads = 1024;
__global__ void __launch_bounds__(kHlJoinThreads)
head_join_kernel(const float4* __restrict__ part, const float* __restrict__ given, const int* __restrict__ tokens, int m, int n, int parts,
                 float* __restrict__ logprob, float* __restrict__ entropy) {
  pdl_wait();
  pdl_trigger();
  __shared__ HlSums sums[kHlJoinThreads / 32][kHlJoinRows];
  const int r = threadIdx.x % kHlJoinRows, group = threadIdx.x / kHlJoinRows, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * kHlJoinRows + r;
  HlSums all = {-INFINITY, 0.f, 0.f};
  constexpr int kGroups = kHlJoinThreads / kHlJoinRows, kAhead = 4;
  for (int i0 = group; i0 < parts; i0 += kAhead * kGroups) {
    float4 v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kGroups;
      v[j] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      if (i < parts && row < m) v[j] = part[static_cast<size_t>(i) * m + row];
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) all.add(v[j].x, v[j].y, v[j].z);
  }
#pragma unroll
  for (int o = 16; o >= kHlJoinRows; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, all.m, o), os = __shfl_xor_sync(0xffffffffu, all.s, o), ow = __shfl_xor_sync(0xffffffffu, all.w, o);
    all.add(om, os, ow);
  }
  if (lane < kHlJoinRows) sums[warp][lane] = all;
  __syncthreads();
  if (threadIdx.x >= kHlJoinRows || row >= m) return;
  for (int w = 1; w < kHlJoinThreads / 32; ++w) all.add(sums[w][r].m, sums[w][r].s, sums[w][r].w);
  const float log_s = log2f(all.s), nan = __int_as_float(0x7fffffff);
  const bool bad = all.s != all.s;
  const int token = tokens[row];
  float lp = nan;
  if (token < 0) {
    lp = 0.f;
  } else if (token < n && !bad) {
    const float x = given[row];
    lp = x > -INFINITY ? (x == all.m ? 0.f : x - all.m) - log_s * kHlLn2 : -INFINITY;
  }
  logprob[row] = lp;
  entropy[row] = bad ? nan : all.m > -INFINITY ? (log_s - all.w / all.s) * kHlLn2 : 0.f;
}

static int head_join(const HlParams& p, int parts, float* logprob, float* entropy, cudaStream_t st) {
  return launch_kernel(head_join_kernel, dim3((p.m + kHlJoinRows - 1) / kHlJoinRows), dim3(kHlJoinThreads), 0, st, 1u, p.part, p.given,
                       p.tokens, p.m, p.n, parts, logprob, entropy) == cudaSuccess
             ? SLLM_OK
             : SLLM_ERR_CUDA;
}

// Allows a kernel its shared memory, once per device (a bit of `known` each).
static bool head_shared_memory(const void* kernel, size_t bytes, std::atomic<uint64_t>& known) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (known.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess) return false;
  known.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

template <int BN>
static int head_logprobs_go(const void* x, const void* w, int k, long long ldx, HlParams& p, float* logprob, float* entropy, cudaStream_t st) {
  using S = HlShape<BN>;
  CUtensorMap tx, tw;
  int rc = cached_kmajor_tmap(&tx, x, 2, p.m, k, ldx * 2, kHlRows);
  if (rc == SLLM_OK) rc = cached_kmajor_tmap(&tw, w, 2, p.n, k, static_cast<long long>(k) * 2, BN / 2);
  if (rc != SLLM_OK) return rc;
  p.tiles_m = (p.m + 255) / 256;
  p.tiles_n = (p.n + BN - 1) / BN;
  const size_t smem = S::kStages * S::kStage + sizeof(HlShared) + 1024;
  static std::atomic<uint64_t> known{0};
  if (!head_shared_memory(reinterpret_cast<const void*>(head_logprobs_kernel<BN>), smem, known)) return SLLM_ERR_CUDA;
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
  if (tiles * p.num_kb > 0x7fffffffLL) return SLLM_ERR_LIMIT;
  const int pairs = tiles < 74 ? static_cast<int>(tiles) : 74;
  if (launch_kernel_cluster(head_logprobs_kernel<BN>, dim3(2 * pairs), dim3(kHlThreads), smem, st, 2u, 1u, tx, tw, p) != cudaSuccess)
    return SLLM_ERR_CUDA;
  return head_join(p, 2 * p.tiles_n, logprob, entropy, st);
}

// CTAs of the kernel for few rows, and the columns of each.
static void head_few_shape(int n, int& ctas, int& share) {
  share = ((n + 147) / 148 + kHfBox - 1) / kHfBox * kHfBox;
  ctas = (n + share - 1) / share;
}

static int head_few_go(const void* x, const void* w, int k, long long ldx, HlParams& p, float* logprob, float* entropy, cudaStream_t st) {
  CUtensorMap tx, tw;
  int x_rows = 8;                           // rows of X that are copied: what lies behind them in shared memory reaches no row that counts
  while (x_rows < p.m) x_rows *= 2;
  int rc = cached_kmajor_tmap(&tx, x, 2, p.m, k, ldx * 2, x_rows);
  if (rc == SLLM_OK) rc = cached_kmajor_tmap(&tw, w, 2, p.n, k, static_cast<long long>(k) * 2, kHfBox);
  if (rc != SLLM_OK) return rc;
  int ctas, share;
  head_few_shape(p.n, ctas, share);
  if ((share / kHfTile + 1LL) * p.num_kb > 0x7fffffffLL) return SLLM_ERR_LIMIT;
  const size_t smem = kHfStages * kHfStage + sizeof(HlShared) + 1024;
  static std::atomic<uint64_t> known{0};
  if (!head_shared_memory(reinterpret_cast<const void*>(head_few_kernel), smem, known)) return SLLM_ERR_CUDA;
  if (launch_kernel(head_few_kernel, dim3(ctas), dim3(kHlThreads), smem, st, 1u, tx, tw, p, share, x_rows) != cudaSuccess) return SLLM_ERR_CUDA;
  return head_join(p, 2 * ctas, logprob, entropy, st);
}

}  // namespace sllm

using namespace sllm;

// Parts of a row: two per tile of bn columns (128 or 256, of CTA pairs), or with bn = 0 two per CTA of the kernel for up to 128 rows.
static long long head_parts(int n, int bn) {
  if (bn) return 2 * ((n + bn - 1LL) / bn);
  int ctas, share;
  head_few_shape(n, ctas, share);
  return 2LL * ctas;
}

// Floats of workspace that m rows take with n tokens.
SLLM_EXPORT long long sllm_head_logprobs_floats(int m, int n, int bn) {
  if (m <= 0 || n <= 0 || n > (1 << 30) || (bn != 0 && bn != 128 && bn != 256)) return 0;
  return m * (4 * head_parts(n, bn) + 1);
}

// x [m, k] bf16 (row stride ldx elements), w [n, k] bf16 contiguous, tokens [m]; logprob and entropy [m].  cap: soft cap (1e-30 to 1e30), or 0.  bn: columns
// of a CTA pair's tile, 128 or 256; 0: the kernel for up to 128 rows.  k a multiple of 8, rows of x multiples of 16 bytes.
SLLM_EXPORT int sllm_head_logprobs(const void* x, const void* w, const int* tokens, int m, int n, int k, long long ldx, float cap, int bn,
                                   float* ws, long long ws_floats, float* logprob, float* entropy, int* status, void* stream) {
  if (!x || !w || !tokens || !ws || !logprob || !entropy || m <= 0 || n <= 0 || k <= 0 || ldx < k ||
      !(cap == 0.f || (cap >= 1e-30f && cap <= 1e30f)))
    return SLLM_ERR_INVALID_ARGUMENT;
  if ((bn != 0 && bn != 128 && bn != 256) || (bn == 0 && m > kHlRows)) return SLLM_ERR_INVALID_ARGUMENT;
  if (m > (1 << 24) || n > (1 << 30) || k > (1 << 24)) return SLLM_ERR_LIMIT;
  if ((k & 7) || (ldx & 7) || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(ws)) & 15))
    return SLLM_ERR_ALIGNMENT;
  if (ws_floats < sllm_head_logprobs_floats(m, n, bn)) return SLLM_ERR_WORKSPACE_TOO_SMALL;
  HlParams p = {};
  p.m = m; p.n = n; p.num_kb = (k + 63) / 64; p.chains = (p.num_kb + kHlChain - 1) / kHlChain;
  p.cap = cap; p.inv_cap = cap > 0.f ? 1.f / cap : 0.f;
  p.tokens = tokens; p.part = reinterpret_cast<float4*>(ws);
  p.given = ws + 4 * head_parts(n, bn) * m;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bn == 0) return head_few_go(x, w, k, ldx, p, logprob, entropy, st);
  return bn == 256 ? head_logprobs_go<256>(x, w, k, ldx, p, logprob, entropy, st) : head_logprobs_go<128>(x, w, k, ldx, p, logprob, entropy, st);
}
