// Log-probabilities of given tokens, the entropy and the largest alternatives of rows of logits:
//   m = max z,  S = sum e^(z - m),  W = sum e^(z - m) (z - m)
//   log p(t) = z_t - m - ln S,   H = -sum p ln p = ln S - W / S
// Alternatives are ordered by logit, equal ones by id.  -inf shuts a token out; a row of nothing else has log p = -inf, H = 0 and
// no alternatives (id -1).  With +inf logits the row is uniform over them; a NaN makes the row's numbers NaN and leaves no
// alternatives.  A given id below 0 stands for no token (0), one beyond the vocabulary has log p NaN.
#include <cfloat>
#include <type_traits>
#include "pair_mma.cuh"
#include "api.h"

namespace sllm {

struct LogprobParams {
  const void* logits;        // rows of `vocab` elements, ld apart
  long long ld;
  int rows, vocab;
  const void* tokens;        // [rows, given] int32 or int64
  int tokens64, given;
  int top;
  float* logprob;            // [rows, given]
  float* entropy;            // [rows]
  int* top_ids;              // [rows, top]
  float* top_logprobs;
};

__device__ __forceinline__ float lp_load(const float* p) { return *p; }
__device__ __forceinline__ float lp_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// 16 bytes of a row, kept as they are loaded.
template <typename T>
struct LpVec {
  static constexpr int kN = 16 / static_cast<int>(sizeof(T));
  uint4 raw;
};
template <typename T>
__device__ __forceinline__ uint32_t lp_shut() {                // -inf in every place of a word
  if constexpr (sizeof(T) == 4) return 0xff800000u;
  else if constexpr (std::is_same_v<T, __half>) return 0xfc00fc00u;
  else return 0xff80ff80u;
}
template <typename T>
__device__ __forceinline__ float lp_max(const LpVec<T>& v) {   // of what is no NaN
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.raw.x), __uint_as_float(v.raw.y)), fmaxf(__uint_as_float(v.raw.z), __uint_as_float(v.raw.w)));
  } else if constexpr (std::is_same_v<T, __half>) {
    const __half2* h = reinterpret_cast<const __half2*>(&v.raw);
    const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.raw);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m.x, m.y);
  }
}
template <typename T>
__device__ __forceinline__ float2 lp_pair(const LpVec<T>& v, int i) {
  if constexpr (sizeof(T) == 4) {
    return i == 0 ? make_float2(__uint_as_float(v.raw.x), __uint_as_float(v.raw.y)) : make_float2(__uint_as_float(v.raw.z), __uint_as_float(v.raw.w));
  } else {
    const uint32_t w = i == 0 ? v.raw.x : i == 1 ? v.raw.y : i == 2 ? v.raw.z : v.raw.w;
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}

// Order of (logit, id) as one integer: larger logits first, then smaller ids; 0 is below every token that is not shut out.
// (x + 0 makes one value of both zeros.)
typedef unsigned long long LpKey;
__device__ __forceinline__ LpKey lp_key(float x, int id) {
  const uint32_t b = __float_as_uint(x + 0.f), o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return x > -INFINITY ? (static_cast<LpKey>(o) << 32) | (0x7fffffffu - static_cast<uint32_t>(id)) : 0ull;
}
__device__ __forceinline__ int lp_key_id(LpKey k) { return static_cast<int>(0x7fffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_value(LpKey k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
// A warp's 32 keys, lane 0 the largest: one exchange of a bitonic network, the whole sort, and the 32 largest of two sorted lists.
__device__ __forceinline__ LpKey lp_exchange(LpKey k, int dist, bool keep_max) {
  const LpKey o = __shfl_xor_sync(0xffffffffu, k, dist);
  return (k > o) == keep_max ? k : o;
}
__device__ __forceinline__ LpKey lp_sort(LpKey k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int dist = size / 2; dist > 0; dist /= 2) k = lp_exchange(k, dist, ((lane & size) == 0) == ((lane & dist) == 0));
  return k;
}
__device__ __forceinline__ LpKey lp_merge(LpKey a, LpKey b) {
  const int lane = threadIdx.x & 31;
  const LpKey r = __shfl_sync(0xffffffffu, b, 31 - lane);
  LpKey k = a > r ? a : r;
#pragma unroll
  for (int dist = 16; dist > 0; dist /= 2) k = lp_exchange(k, dist, (lane & dist) == 0);
  return k;
}

__device__ __forceinline__ float lp_exp2(float x) {            // 0 below the smallest normal number
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpFloor = -200.f;         // differences below it count as it: e^-200 is 0 in fp32, and 0 times it is no NaN
constexpr float kLpSlack = 4.f;            // a thread's sums are taken anew when a logit passes their reference by more
constexpr int kLpMaxCluster = 8;
constexpr int kLpSmallUnits = 1024;
constexpr int kLpFill = 592;
constexpr int kLpMaxVocab = 1 << 30;       // ids and units stay below 2^31

// Sums of one part of a row: reference m, S and W as above with respect to it.
struct LpStats {
  float m, s, w;
  __device__ __forceinline__ void rebase(float to) {           // to >= m
    const float d = fmaxf(m - to, kLpFloor), e = lp_exp2(d * kLpLog2e);
    w = e * (w + d * s);
    s *= e;
    m = to;
  }
};

template <int kThreads>
struct __align__(16) LpShared {
  static constexpr int kWarps = kThreads / 32;
  LpStats stat[kWarps];
  float best[kWarps];
  LpKey list[kWarps][32];
  LpKey found[32];
  int count;
  LpStats part[kLpMaxCluster];             // of the first CTA: what the CTAs of a row found
  float part_best[kLpMaxCluster];
  LpKey part_list[kLpMaxCluster][32];
  int bad[2];
};

// A cluster of CTAs per row (one where there are many rows), each with a range of the row's 16-byte units; unit v of a range goes to
// thread v mod kThreads.  One pass takes S and W per thread with respect to a reference that follows the maximum loosely, so that the
// usual unit has no branch, and the thread's largest logit.
// Alternatives: the top-th largest of the threads' maxima bounds the wanted ones from below, and only as many threads have
// logits above it as there are alternatives; those threads' units are read again (out of L2) and what passes the bound is sorted by one warp.
// Where more than 32 pass it (runs of equal or ordered logits), sorted lists are merged 32 at a time instead.
template <typename T, int kThreads, bool kTop>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobParams p, int cluster) {
  constexpr int kN = LpVec<T>::kN, kWarps = kThreads / 32, kAhead = 4;
  __shared__ LpShared<kThreads> sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int rank = cluster > 1 ? static_cast<int>(blockIdx.x % cluster) : 0;
  const long long row = blockIdx.x / cluster;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_trigger();
  const T* z = static_cast<const T*>(p.logits) + row * p.ld;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));      // elements of the first unit ahead of the row
  const uint4* units = reinterpret_cast<const uint4*>(z - shift);
  const int n_units = static_cast<int>((static_cast<long long>(shift) + p.vocab + kN - 1) / kN);
  const int per = (n_units + cluster - 1) / cluster, lo = min(rank * per, n_units), hi = min(lo + per, n_units);
  // whole units: neither the first one with a shift nor a last one that is not full
  const int whole_lo = shift ? 1 : 0, whole_hi = static_cast<int>((static_cast<long long>(shift) + p.vocab) / kN);
  constexpr float kNone = -INFINITY;

  // any unit, places outside the row shut out
  auto load_unit = [&](int v) {
    LpVec<T> u;
    if (v >= whole_lo && v < whole_hi) {
      u.raw = units[v];
    } else {
      u.raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
      T* e = reinterpret_cast<T*>(&u.raw);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const long long id = static_cast<long long>(v) * kN + i - shift;
        if (id >= 0 && id < p.vocab) e[i] = z[id];
      }
    }
    return u;
  };
  // the given tokens' logits, ahead of the pass
  const float nan = __int_as_float(0x7fffffff);
  auto given = [&](int j, long long& id) {
    const long long at = row * p.given + j;
    id = p.tokens64 ? static_cast<const long long*>(p.tokens)[at] : static_cast<const int*>(p.tokens)[at];
    return id >= 0 && id < p.vocab ? lp_load(z + id) : 0.f;
  };
  long long tok = -1;
  float tok_x = 0.f;
  if (rank == 0 && tid < p.given) tok_x = given(tid, tok);

  LpStats st = {-FLT_MAX, 0.f, 0.f};
  float best = kNone;
  int best_at = 0;
  uint64_t s2 = 0ull, w2 = 0ull;
  auto add = [&](const LpVec<T>& u, int v) {
    const float top = lp_max(u);
    if constexpr (kTop) best_at = top > best ? v : best_at;
    best = fmaxf(best, top);
    if (top > st.m + kLpSlack) {
      const float2 s = unpack_f32x2(s2), w = unpack_f32x2(w2);
      st.s = s.x + s.y;
      st.w = w.x + w.y;
      st.rebase(top);
      s2 = pack_f32x2(st.s, 0.f);
      w2 = pack_f32x2(st.w, 0.f);
    }
    const uint64_t ref = pack_f32x2(-st.m, -st.m), scale = pack_f32x2(kLpLog2e, kLpLog2e);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const float2 x = lp_pair(u, i);
      float2 d = unpack_f32x2(lp_add2(pack_f32x2(x.x, x.y), ref));
      const uint64_t d2 = pack_f32x2(lp_max_nan(d.x, kLpFloor), lp_max_nan(d.y, kLpFloor));
      const float2 t = unpack_f32x2(mul_f32x2(d2, scale));
      const uint64_t e2 = pack_f32x2(lp_exp2(t.x), lp_exp2(t.y));
      s2 = lp_add2(s2, e2);
      w2 = fma_f32x2(e2, d2, w2);
    }
  };
  if (lo + tid < min(hi, whole_lo)) add(load_unit(lo + tid), lo + tid);
  // (whole_lo is at most 1: only thread 0 of the first range has such a unit, and goes on behind it)
  const int end = min(hi, whole_hi);
  for (int v = lo + tid + (lo + tid < whole_lo ? kThreads : 0); v < end; v += kAhead * kThreads) {
    LpVec<T> u[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      u[i].raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
      if (v + i * kThreads < end) u[i].raw = units[v + i * kThreads];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(u[i], v + i * kThreads);
  }
  {
    const int v = n_units - 1;                                 // the last unit, where it is not whole and was not the first as well
    if (v >= whole_hi && v >= whole_lo && v >= lo && v < hi && (v - lo) % kThreads == tid) add(load_unit(v), v);
  }

  // the CTA's sums
  {
    const float2 s = unpack_f32x2(s2), w = unpack_f32x2(w2);
    st.s = s.x + s.y;
    st.w = w.x + w.y;
  }
  const float warp_best = warp_max(best);
  if (lane == 0) sh.best[warp] = warp_best;
  if (tid == 0) sh.bad[0] = sh.bad[1] = sh.count = 0;
  __syncthreads();
  float all_best = sh.best[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) all_best = fmaxf(all_best, sh.best[w]);
  const bool odd = !(all_best < INFINITY) || st.s != st.s;     // +inf or NaN among the logits
  if (__syncthreads_or(odd)) {
    int inf = 0, bad = 0;
    for (int v = lo + tid; v < hi; v += kThreads) {
      const LpVec<T> u = load_unit(v);
#pragma unroll
      for (int i = 0; i < kN / 2; ++i) {
        const float2 x = lp_pair(u, i);
        inf += (x.x == INFINITY) + (x.y == INFINITY);
        bad += (x.x != x.x) + (x.y != x.y);
      }
    }
    if (inf) atomicAdd(&sh.bad[0], inf);
    if (bad) atomicAdd(&sh.bad[1], bad);
    __syncthreads();
    // uniform over +inf: every one counts 1, with no difference to the maximum
    st.m = all_best;
    st.s = tid == 0 ? (sh.bad[1] ? nan : static_cast<float>(sh.bad[0])) : 0.f;
    st.w = 0.f;
  } else {
    st.rebase(fmaxf(all_best, -FLT_MAX));
  }
  st.s = warp_sum(st.s);
  st.w = warp_sum(st.w);
  if (lane == 0) sh.stat[warp] = st;
  __syncthreads();
  LpStats mine = sh.stat[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    mine.s += sh.stat[w].s;
    mine.w += sh.stat[w].w;
  }

  LpKey key = 0;                                               // lane i of warp 0: the CTA's i-th alternative
  if constexpr (kTop) {
    // the thread's maximum stands for the last place of its unit, which orders it rightly against other units
    key = lp_sort(lp_key(best, best_at * kN + kN - 1 - shift));
#pragma unroll
    for (int half = kWarps / 2; half > 0; half /= 2) {
      if (warp >= half && warp < 2 * half) sh.list[warp][lane] = key;
      __syncthreads();
      if (warp < half) key = lp_merge(key, sh.list[warp + half][lane]);
    }
    if (warp == 0) sh.found[lane] = lane < p.top ? key : 0;
    __syncthreads();
    const LpKey bound = sh.found[p.top - 1];                   // 0: every token counts
    LpKey mine_k = 0;
    // what passes the bound among a winner's units, one place of the units at a time
    auto scan = [&](auto&& take) {
      for (int j = warp; j < p.top; j += kWarps) {
        const LpKey win = sh.found[j];
        if (!win) break;
        const int owner = ((lp_key_id(win) - (kN - 1) + shift) / kN - lo) % kThreads;
        for (int v0 = lo + owner; v0 < hi; v0 += 32 * kThreads) {
          const int v = v0 + lane * kThreads;
          LpVec<T> u;
          u.raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
          if (v < hi) u = load_unit(v);
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const float2 x = lp_pair(u, i / 2);
            const LpKey k = lp_key(i & 1 ? x.y : x.x, v * kN + i - shift);
            take(k >= bound ? k : 0);
          }
        }
      }
    };
    LpKey* pool = &sh.list[0][0];                              // 32 keys at least
    scan([&](LpKey k) {
      if (k) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < 32) pool[at] = k;
      }
    });
    __syncthreads();
    if (sh.count <= 32) {
      if (warp == 0) key = lp_sort(lane < sh.count ? pool[lane] : 0);
    } else {
      scan([&](LpKey k) {
        const LpKey least = __shfl_sync(0xffffffffu, mine_k, 31);
        if (__any_sync(0xffffffffu, k > least)) mine_k = lp_merge(mine_k, lp_sort(k));
      });
      __syncthreads();
      key = mine_k;
#pragma unroll
      for (int half = kWarps / 2; half > 0; half /= 2) {
        if (warp >= half && warp < 2 * half) sh.list[warp][lane] = key;
        __syncthreads();
        if (warp < half) key = lp_merge(key, sh.list[warp + half][lane]);
      }
    }
  }

  if (cluster > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");          // the first CTA runs
    uint32_t to;
    if (kTop && warp == 0) {
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(&sh.part_list[rank][lane])));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
    }
    if (tid == 0) {
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(&sh.part[rank])));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(mine.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(mine.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(mine.w) : "memory");
    }
    __syncwarp();
    cluster_sync_pair();
    if (rank != 0) return;
    float m = sh.part[0].m;
    for (int c = 1; c < cluster; ++c) m = fmaxf(m, sh.part[c].m);
    mine = {m, 0.f, 0.f};
    for (int c = 0; c < cluster; ++c) {
      LpStats q = sh.part[c];
      if (q.m == m) {                                          // (+inf: the parts without one have nothing to add)
        mine.s += q.s;
        mine.w += q.w;
      } else {
        q.rebase(m);
        mine.s += q.s;                                         // a NaN of any part passes through
        mine.w += q.w;
      }
    }
    if (kTop && warp == 0) {
      key = sh.part_list[0][lane];
      for (int c = 1; c < cluster; ++c) key = lp_merge(key, sh.part_list[c][lane]);
    }
  }
  const float ln_s = logf(mine.s);
  const bool bad = mine.s != mine.s;
  auto logp = [&](float x) { return bad ? nan : x > -INFINITY ? (x == mine.m ? 0.f : x - mine.m) - ln_s : -INFINITY; };
  if (tid == 0) p.entropy[row] = bad ? nan : mine.s > 0.f ? ln_s - mine.w / mine.s : 0.f;
  for (int j = tid; j < p.given; j += kThreads) {
    if (j != tid) tok_x = given(j, tok);
    p.logprob[row * p.given + j] = tok < 0 ? 0.f : tok >= p.vocab ? nan : logp(tok_x);
  }
  if (kTop && warp == 0 && lane < p.top) {
    p.top_ids[row * p.top + lane] = key && !bad ? lp_key_id(key) : -1;
    p.top_logprobs[row * p.top + lane] = bad ? nan : key ? logp(lp_key_value(key)) : -INFINITY;
  }
}

template <typename T, int kThreads>
static cudaError_t logprobs_go(const LogprobParams& p, int cluster, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.rows) * cluster), block(kThreads);
  return p.top ? launch_kernel_cluster(logprobs_kernel<T, kThreads, true>, grid, block, 0, st, cluster, 1u, p, cluster)
               : launch_kernel_cluster(logprobs_kernel<T, kThreads, false>, grid, block, 0, st, cluster, 1u, p, cluster);
}

template <typename T>
static cudaError_t logprobs_go(const LogprobParams& p, cudaStream_t st) {
  const long long units = (static_cast<long long>(p.vocab) + LpVec<T>::kN - 1) / LpVec<T>::kN;
  if (units <= kLpSmallUnits) return logprobs_go<T, 64>(p, 1, st);
  int cluster = 1;
  while (cluster < kLpMaxCluster && static_cast<long long>(p.rows) * cluster * 2 <= kLpFill && units >= 2 * cluster * 256) cluster *= 2;
  return logprobs_go<T, 256>(p, cluster, st);
}

}  // namespace sllm

using namespace sllm;

// logits [rows, vocab] of dtype 0 bf16, 1 fp16, 2 fp32, rows ld elements apart; tokens [rows, given] int32 (tokens64: int64);
// logprob [rows, given], entropy [rows], top_ids / top_logprobs [rows, top] (0 to 32, null with 0).
SLLM_EXPORT int sllm_token_logprobs(const void* logits, long long ld, int rows, int vocab, int dtype, const void* tokens, int tokens64,
                                    int given, int top, float* logprob, float* entropy, int* top_ids, float* top_logprobs, void* stream) {
  if (!logits || rows <= 0 || vocab <= 0 || ld < 0 || given < 0 || top < 0 || !entropy || dtype < 0 || dtype > 2) return SLLM_ERR_INVALID_ARGUMENT;
  if ((given && (!tokens || !logprob)) || (top && (!top_ids || !top_logprobs))) return SLLM_ERR_INVALID_ARGUMENT;
  if (top > 32 || vocab > kLpMaxVocab) return SLLM_ERR_LIMIT;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return SLLM_ERR_ALIGNMENT;
  LogprobParams p = {logits, ld, rows, vocab, tokens, tokens64, given, top, logprob, entropy, top_ids, top_logprobs};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == 0 ? logprobs_go<__nv_bfloat16>(p, st) : dtype == 1 ? logprobs_go<__half>(p, st) : logprobs_go<float>(p, st);
  return e == cudaSuccess ? SLLM_OK : SLLM_ERR_CUDA;
}
