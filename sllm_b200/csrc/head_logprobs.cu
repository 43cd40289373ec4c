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
// A tile's sum over K is taken in chains of kHlChain K blocks with an accumulator of their own, which the epilogue warps add in fp32
// registers while the next chain is multiplied: tensor memory rounds towards zero, and a chain's error grows with its length.
// Few rows need no tile of their own: rows beyond the last are filled with zeros, cost no reading, and their products run beside the
// reading of W.
#include <cfloat>
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
      if (p.cap > 0.f) {
#pragma unroll
        for (int c = 0; c < S::kCols; ++c) z[c] = p.cap * tanhf(z[c] * p.inv_cap);
      }
      if (__any_sync(0xffffffffu, token >= n0 && token < n0 + S::kCols)) {
        float x = 0.f;
#pragma unroll
        for (int c = 0; c < S::kCols; ++c) x = token - n0 == c ? z[c] : x;
        if (token >= n0 && token < min(n0 + S::kCols, p.n)) p.given[row] = x;
      }
      if (n0 + S::kCols > p.n) {                           // tokens beyond the last
#pragma unroll
        for (int c = 0; c < S::kCols; ++c) z[c] = n0 + c < p.n ? z[c] : -INFINITY;
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < S::kCols; c += 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) m4[i] = fmaxf(m4[i], z[c + i]);
      const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
      if (m < INFINITY) {
        const float ref = m > -INFINITY ? m : 0.f;         // (nothing but -inf: every term is 2^-1000)
#pragma unroll
        for (int c = 0; c < S::kCols; c += 2) {
          const float t0 = hl_max_nan((z[c] - ref) * kHlLog2e, -1000.f), t1 = hl_max_nan((z[c + 1] - ref) * kHlLog2e, -1000.f);
          const float e0 = hl_exp2(t0), e1 = hl_exp2(t1);
          s0 += e0;
          s1 += e1;
          w0 = fmaf(e0, t0, w0);
          w1 = fmaf(e1, t1, w1);
        }
      } else {                                             // uniform over +inf
#pragma unroll
        for (int c = 0; c < S::kCols; ++c) s0 += z[c] != z[c] ? z[c] : z[c] == INFINITY ? 1.f : 0.f;
      }
      if (row < p.m) p.part[static_cast<size_t>(2 * tn + grp) * p.m + row] = make_float4(m, s0 + s1, w0 + w1, 0.f);
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

// The parts of a row: eight rows per CTA, so that a line of parts is read as a whole, 128 threads for each.
constexpr int kHlJoinRows = 8, kHlJoinThreads = 1024;
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
  if (cudaFuncSetAttribute(head_logprobs_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return SLLM_ERR_CUDA;
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
  if (tiles * p.num_kb > 0x7fffffffLL) return SLLM_ERR_LIMIT;
  const int pairs = tiles < 74 ? static_cast<int>(tiles) : 74;
  if (launch_kernel_cluster(head_logprobs_kernel<BN>, dim3(2 * pairs), dim3(kHlThreads), smem, st, 2u, 1u, tx, tw, p) != cudaSuccess)
    return SLLM_ERR_CUDA;
  return launch_kernel(head_join_kernel, dim3((p.m + kHlJoinRows - 1) / kHlJoinRows), dim3(kHlJoinThreads), 0, st, 1u, p.part, p.given,
                       p.tokens, p.m, p.n, 2 * p.tiles_n, logprob, entropy) == cudaSuccess
             ? SLLM_OK
             : SLLM_ERR_CUDA;
}

}  // namespace sllm

using namespace sllm;

// Floats of workspace that m rows take with n tokens.
SLLM_EXPORT long long sllm_head_logprobs_floats(int m, int n, int bn) {
  if (m <= 0 || n <= 0 || (bn != 128 && bn != 256)) return 0;
  return static_cast<long long>(m) * (8LL * ((n + bn - 1LL) / bn) + 1);
}

// x [m, k] bf16 (row stride ldx elements), w [n, k] bf16 contiguous, tokens [m]; logprob and entropy [m].  cap > 0: soft cap.  bn: columns
// of a pair's tile, 128 or 256.  k a multiple of 8, rows of x multiples of 16 bytes.
SLLM_EXPORT int sllm_head_logprobs(const void* x, const void* w, const int* tokens, int m, int n, int k, long long ldx, float cap, int bn,
                                   float* ws, long long ws_floats, float* logprob, float* entropy, int* status, void* stream) {
  if (!x || !w || !tokens || !ws || !logprob || !entropy || m <= 0 || n <= 0 || k <= 0 || ldx < k || !(cap >= 0.f && cap < INFINITY))
    return SLLM_ERR_INVALID_ARGUMENT;
  if (bn != 128 && bn != 256) return SLLM_ERR_INVALID_ARGUMENT;
  if (m > (1 << 24) || n > (1 << 30) || k > (1 << 24)) return SLLM_ERR_LIMIT;
  if ((k & 7) || (ldx & 7) || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(ws)) & 15))
    return SLLM_ERR_ALIGNMENT;
  if (ws_floats < sllm_head_logprobs_floats(m, n, bn)) return SLLM_ERR_WORKSPACE_TOO_SMALL;
  HlParams p = {};
  p.m = m; p.n = n; p.num_kb = (k + 63) / 64; p.chains = (p.num_kb + kHlChain - 1) / kHlChain;
  p.cap = cap; p.inv_cap = cap > 0.f ? 1.f / cap : 0.f;
  p.tokens = tokens; p.part = reinterpret_cast<float4*>(ws);
  p.given = ws + static_cast<long long>(m) * 8 * ((n + bn - 1) / bn);
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return bn == 256 ? head_logprobs_go<256>(x, w, k, ldx, p, logprob, entropy, st) : head_logprobs_go<128>(x, w, k, ldx, p, logprob, entropy, st);
}
