// Log-probabilities of given tokens, the entropy and the largest alternatives of rows of logits:
//   m = max z,  S = sum e^(z - m),  W = sum e^(z - m) (z - m)
//   log p(t) = z_t - m - ln S,   H = -sum p ln p = ln S - W / S
// Alternatives are ordered by logit, equal ones by id.  -inf shuts a token out; a row of nothing else has log p = -inf, H = 0 and
// no alternatives (id -1).  With +inf logits the row is uniform over them; a NaN makes the row's numbers NaN and leaves no
// alternatives.  A given id below 0 stands for no token (0), one beyond the vocabulary has log p NaN.
#include <algorithm>
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
__device__ __forceinline__ uint32_t lp_word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
template <typename T>
__device__ __forceinline__ float2 lp_split(uint32_t w) {       // of 16-bit types
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ float2 lp_pair(const LpVec<T>& v, int i) {
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(lp_word(v.raw, 2 * i)), __uint_as_float(lp_word(v.raw, 2 * i + 1)));
  else return lp_split<T>(lp_word(v.raw, i));
}

// Sums are taken in powers of two, t = z log2(e) - m2 with m2 the rounded product of the reference: S = sum 2^t and W = sum 2^t t.
// Rounding moves m2 by up to half a unit in its last place (`lp_rest`), and 2^t of the largest logit is 2 to as much: between 1/2 and 2 below
// 2^24, but 0 or infinite from 1e10 on.  So logits below kLow count as it (-inf too, whose 2^t t would be NaN), and where a range's
// largest logit is not well above kLow, or beyond kHigh, its sums are taken anew from exact differences (`lp_wide`): the range is read
// twice (4096 x 128256 bf16 about 1e8: 514 us, 184 of ordinary logits; one such row 6.9 and 3.7).
template <typename T>
struct LpRange {
  static constexpr bool kHalf = std::is_same_v<T, __half>;
  static constexpr float kLow = kHalf ? -60000.f : -16777216.f;         // (-2^24)
  static constexpr float kWide = kHalf ? -59000.f : -8388608.f;         // (-2^23)
  static constexpr float kHigh = 8388608.f;
  static constexpr uint32_t kLowPair = kHalf ? 0xfb53fb53u : 0xcb80cb80u;
};
template <typename T>
__device__ __forceinline__ bool lp_wide(float m) { return !(m > LpRange<T>::kWide && m < LpRange<T>::kHigh); }
constexpr float kLpLog2e = 1.4426950408889634f, kLpLn2 = 0.6931471805599453f;
template <typename T>
__device__ __forceinline__ float lp_rest(float m) {            // m log2(e) less the reference of a range's sums with this maximum
  return lp_wide<T>(m) ? 0.f : fmaf(m, kLpLog2e, -__fmul_rn(m, kLpLog2e));
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 lp_pair_from_low(const LpVec<T>& v, int i) {      // lp_pair, nothing below kLow
  if constexpr (sizeof(T) == 4) {
    const float2 x = lp_pair(v, i);
    return make_float2(lp_max_nan(x.x, LpRange<T>::kLow), lp_max_nan(x.y, LpRange<T>::kLow));
  } else {
    uint32_t w;
    if constexpr (LpRange<T>::kHalf) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(w) : "r"(lp_word(v.raw, i)), "r"(LpRange<T>::kLowPair));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(w) : "r"(lp_word(v.raw, i)), "r"(LpRange<T>::kLowPair));
    return lp_split<T>(w);
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
// (Floats hold no NaN.)
__device__ __forceinline__ LpKey lp_exchange(LpKey k, int dist, bool keep_max) {
  const LpKey o = __shfl_xor_sync(0xffffffffu, k, dist);
  return (k > o) == keep_max ? k : o;
}
__device__ __forceinline__ float lp_exchange(float k, int dist, bool keep_max) {
  const float o = __shfl_xor_sync(0xffffffffu, k, dist);
  return keep_max ? fmaxf(k, o) : fminf(k, o);
}
template <typename K>
__device__ __forceinline__ K lp_sort(K k) {
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
// A load that stays where it is written, so that several are under way at a time; the row passes L1 by.
__device__ __forceinline__ uint4 lp_stream(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

constexpr float kLpSlack = 4.f;            // a thread's sums are taken anew when a logit passes their reference by more

constexpr int kLpMaxCluster = 8;
constexpr int kLpSmallUnits = 1024;
constexpr int kLpFill = 592;                // CTAs of 256 threads that the card holds; of 128 threads twice as many
constexpr int kLpLongRows = 2368;
constexpr int kLpMaxVocab = 1 << 30;       // ids and units stay below 2^31

// Sums of one part of a row with respect to m.
struct LpStats {
  float m, s, w;
  __device__ __forceinline__ void shift(float t) {             // by 2^t, t <= 0 and finite
    const float e = lp_exp2(t);
    w = e * fmaf(t, s, w);
    s *= e;
  }
  __device__ __forceinline__ void add(const LpStats& o) {      // (of the same m; NaN passes through)
    s += o.s;
    w += o.w;
  }
  __device__ __forceinline__ LpStats at(float max, float t) const {
    LpStats r = *this;
    if (m == max) return r;
    r.m = max;
    r.shift(fmaxf(t, -1000.f));
    return r;
  }
  // A warp's sums, which refer to a rounded product whatever its maximum, with respect to the maximum of a range that is not wide ...
  template <typename T>
  __device__ __forceinline__ LpStats in_range(float max) const {
    return at(max, __fmul_rn(fmaxf(m, LpRange<T>::kLow), kLpLog2e) - __fmul_rn(max, kLpLog2e));
  }
  // ... and a range's with respect to the row's, either of which may be.
  template <typename T>
  __device__ __forceinline__ LpStats in_row(float max) const {
    if (lp_wide<T>(m) || lp_wide<T>(max)) return at(max, (m - max) * kLpLog2e + (lp_rest<T>(max) - lp_rest<T>(m)));
    return at(max, __fmul_rn(m, kLpLog2e) - __fmul_rn(max, kLpLog2e));
  }
};

constexpr int kLpParts = 4;                // of a range, with a maximum per thread each
constexpr int kLpPool = 256;               // candidates that are ranked against one another

template <int kThreads, int kParts>
struct __align__(16) LpShared {
  static constexpr int kWarps = kThreads / 32;
  LpStats stat[kWarps];
  float high[32];                          // the largest of the threads' maxima of each warp
  int wins, count;
  float best[kParts][kThreads];            // the largest logit of a thread's units by part of the range
  unsigned short win[kParts * kThreads];   // parts with logits at or above the bound: part kThreads + thread
  LpKey pool[kLpPool];
  LpKey merged[kWarps][32];
  LpKey list[32];                          // the CTA's alternatives
  LpStats part[kLpMaxCluster];             // of the first CTA: what the CTAs of a row found
  LpKey part_list[kLpMaxCluster][32];
  int inf, nan;
};

// A cluster of CTAs per row (one where there are many rows), each with a range of the row's 16-byte units; unit v of a range goes to
// thread v mod kThreads.  One pass takes S and W per thread with respect to a reference that follows the maximum loosely, so that the
// usual unit has no branch, and the thread's largest logit.
// Alternatives: the top-th largest of the threads' maxima bounds the wanted ones from below, and hardly more parts of threads' units have
// logits at or above it than there are alternatives; those units are read again (out of L2) and what passes the bound is ranked by
// counting.  Where more than kLpPool logits pass it (runs of equal or ordered ones), sorted lists are merged 32 at a time instead.
// What bounds it: memory and the exponentials together for many rows (4096 x 128256 bf16, 162.5 us at the copy bandwidth: 171 to 187 from one
// process to the next, 178 under the profiler with 0.72 of the DRAM's peak, 0.74 of the exponential unit and 0.62 of the issue slots busy;
// 1500 x 32768 fp16: 23.2 of 15.2, rows start and end too often), for few the chain of a row (one of 128256: 3.7 us, 7.0 with 20 alternatives,
// of which the launch takes 2).
// kLong, for many long rows: rounds of loads without a bound, and the maxima of kLpParts parts of a thread's units, so that less is read
// again (4096 x 128256 bf16, us, both forms in one process: without alternatives 190 -> 184, 5 of them 214 -> 207, 32 of them 316 -> 257;
// with 700 rows 5 take 43.5 -> 45.3).
template <typename T, int kThreads, bool kTop, bool kLong>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprobs_kernel(const LogprobParams p, int cluster) {
  constexpr int kN = LpVec<T>::kN, kWarps = kThreads / 32, kAhead = 4, kParts = kLong ? kLpParts : 1;
  __shared__ LpShared<kThreads, kParts> sh;
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
  // the given tokens: ids ahead of the pass, their logits behind it
  const float nan = __int_as_float(0x7fffffff);
  auto token = [&](int j) {
    const long long at = row * p.given + j;
    return p.tokens64 ? static_cast<const long long*>(p.tokens)[at] : static_cast<long long>(static_cast<const int*>(p.tokens)[at]);
  };
  auto logit = [&](long long id) { return id >= 0 && id < p.vocab ? lp_load(z + id) : 0.f; };
  long long tok = -1;
  if (rank == 0 && tid < p.given) tok = token(tid);

  float best = kNone;                                          // the thread's largest logit
  float limit = LpRange<T>::kLow, m2 = LpRange<T>::kLow * kLpLog2e;      // reference of its sums, as the logit that asks for another one and as m2
  uint64_t s2 = 0ull, w2 = 0ull;
  auto add = [&](const LpVec<T>& u) {
    const float top = lp_max(u);
    best = fmaxf(best, top);
    if (top > limit) {
      const float2 s = unpack_f32x2(s2), w = unpack_f32x2(w2);
      const float next = top * kLpLog2e;
      LpStats st = {0.f, s.x + s.y, w.x + w.y};
      st.shift(m2 - next);
      s2 = pack_f32x2(st.s, 0.f);
      w2 = pack_f32x2(st.w, 0.f);
      m2 = next;
      limit = top + kLpSlack;
    }
    const uint64_t ref = pack_f32x2(-m2, -m2), scale = pack_f32x2(kLpLog2e, kLpLog2e);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const float2 x = lp_pair_from_low(u, i);
      const uint64_t t2 = fma_f32x2(pack_f32x2(x.x, x.y), scale, ref);
      const float2 t = unpack_f32x2(t2);
      const uint64_t e2 = pack_f32x2(lp_exp2(t.x), lp_exp2(t.y));
      s2 = add_f32x2(s2, e2);
      w2 = fma_f32x2(e2, t2, w2);
    }
  };
  const int each = (hi - lo + kThreads - 1) / kThreads;        // units per thread; per part, in whole rounds of loads
  const int part_units = kParts > 1 ? max((each + kParts * kAhead - 1) / (kParts * kAhead), 1) * kAhead : max(each, 1);
  if (lo + tid < min(hi, whole_lo)) add(load_unit(lo + tid));
  // (whole_lo is at most 1: only thread 0 of the first range has such a unit, and goes on behind it)
  const int end = min(hi, whole_hi);
  int v = lo + tid + (lo + tid < whole_lo ? kThreads : 0);
  if constexpr (!kLong) {
    for (; v < end; v += kAhead * kThreads) {
      LpVec<T> u[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        u[i].raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
        if (v + i * kThreads < end) u[i].raw = lp_stream(units + v + i * kThreads);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) add(u[i]);
    }
  } else {
#pragma unroll 1
    for (int part = 0; part < kParts; ++part) {
      const int stop = min(end, lo + (part + 1) * part_units * kThreads);
      for (; v + (kAhead - 1) * kThreads < stop; v += kAhead * kThreads) {
        LpVec<T> u[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) u[i].raw = lp_stream(units + v + i * kThreads);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) add(u[i]);
      }
      if (v < stop) {
        LpVec<T> u[kAhead - 1];
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) {
          u[i].raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
          if (v + i * kThreads < stop) u[i].raw = lp_stream(units + v + i * kThreads);
        }
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) add(u[i]);
      }
      v = lo + tid + (part + 1) * part_units * kThreads;       // (a thread that began one unit later goes on with the others)
      sh.best[part][tid] = best;
      if (kTop) best = kNone;
    }
  }
  {
    const int v = n_units - 1;                                 // the last unit, where it is not whole and was not the first as well
    if (v >= whole_hi && v >= whole_lo && v >= lo && v < hi && (v - lo) % kThreads == tid) {
      add(load_unit(v));
      if constexpr (kTop && kLong) {
        float& its = sh.best[(v - lo) / kThreads / part_units][tid];
        its = fmaxf(its, best);
      }
    }
  }
  if constexpr (kTop && kLong) {
#pragma unroll
    for (int part = 0; part < kParts; ++part) best = fmaxf(best, sh.best[part][tid]);
  }

  float tok_x = logit(tok);

  // the CTA's sums: the threads' of each warp with respect to the warp's maximum, then the warps'
  auto join = [&](const LpStats* part, int parts, auto to) {
    float m = part[0].m;
    for (int i = 1; i < parts; ++i) m = fmaxf(m, part[i].m);
    LpStats all = {m, 0.f, 0.f};
    for (int i = 0; i < parts; ++i) all.add(to(part[i], m));
    return all;
  };
  {
    const float2 s = unpack_f32x2(s2), w = unpack_f32x2(w2);
    LpStats st = {warp_max(best), s.x + s.y, w.x + w.y};
    // (a warp without logits above kLow leaves a sum that `in_range` takes away; t is large only where the range is taken anew)
    st.shift(m2 - __fmul_rn(fmaxf(st.m, LpRange<T>::kLow), kLpLog2e));
    st.s = warp_sum(st.s);
    st.w = warp_sum(st.w);
    if (lane == 0) sh.stat[warp] = st;
    if (tid == 0) sh.inf = sh.nan = sh.count = sh.wins = 0;
  }
  __syncthreads();
  bool again = false;
  {
    float m = kNone;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      m = fmaxf(m, sh.stat[w].m);
      again |= !(sh.stat[w].s < INFINITY);
    }
    if (lp_wide<T>(m)) again = true;
  }
  LpStats mine;
  if (!again) {
    mine = join(sh.stat, kWarps, [](const LpStats& s, float max) { return s.in_range<T>(max); });
  } else {
    float m = sh.stat[0].m;
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh.stat[w].m);
    LpStats st = {m, 0.f, 0.f};
    int inf = 0, bad = 0;
    for (int v = lo + tid; v < hi; v += kThreads) {
      const LpVec<T> u = load_unit(v);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float2 x = lp_pair(u, i / 2);
        const float y = i & 1 ? x.y : x.x;
        inf += y == INFINITY;
        bad += y != y;
        if (y > -INFINITY && m < INFINITY) {
          const float t = fmaxf((y == m ? 0.f : y - m) * kLpLog2e, -1000.f), e = lp_exp2(t);
          st.s += e;
          st.w += e * t;
        }
      }
    }
    st.s = warp_sum(st.s);
    st.w = warp_sum(st.w);
    inf = __reduce_add_sync(0xffffffffu, inf);
    bad = __reduce_add_sync(0xffffffffu, bad);
    __syncthreads();
    if (lane == 0) {
      sh.stat[warp] = st;
      atomicAdd(&sh.inf, inf);
      atomicAdd(&sh.nan, bad);
    }
    __syncthreads();
    mine = {m, 0.f, 0.f};
    for (int w = 0; w < kWarps; ++w) mine.add(sh.stat[w]);
    if (sh.inf) mine = {m, static_cast<float>(sh.inf), 0.f};   // uniform over +inf
    if (sh.nan) mine.s = nan;
  }

  if constexpr (kTop) {
    // the bound: top-th largest among the first 32 / kWarps maxima of each warp, which leaves hardly more than the wanted ones above it
    constexpr int kHigh = 32 / kWarps;
    const float v = lp_sort(best);
    if (lane < kHigh) sh.high[warp * kHigh + lane] = v;
    __syncthreads();
    const float bound = __shfl_sync(0xffffffffu, lp_sort(sh.high[lane]), p.top - 1);      // -inf: every token counts
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const float x = kLong ? sh.best[part][tid] : best;
      if (x >= bound && x > -INFINITY) sh.win[atomicAdd(&sh.wins, 1)] = static_cast<unsigned short>(part * kThreads + tid);
    }
    __syncthreads();
    // their units, dealt out over all threads
    const int todo = sh.wins * part_units;
    auto unit_of = [&](int i) {                                // beyond the range: none
      if (i >= todo) return hi;
      const int win = sh.win[i / part_units];
      return lo + win % kThreads + (win / kThreads * part_units + i % part_units) * kThreads;
    };
    for (int i0 = tid; i0 < todo; i0 += kAhead * kThreads) {
      LpVec<T> u[kAhead];
      int at[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        at[i] = unit_of(i0 + i * kThreads);
        u[i].raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
        if (at[i] < hi) u[i] = load_unit(at[i]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (!(lp_max(u[i]) >= bound)) continue;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float2 x = lp_pair(u[i], e / 2);
          const float y = e & 1 ? x.y : x.x;
          if (y >= bound && y > -INFINITY) {
            const int n = atomicAdd(&sh.count, 1);
            if (n < kLpPool) sh.pool[n] = lp_key(y, at[i] * kN + e - shift);
          }
        }
      }
    }
    if (tid < 32) sh.list[tid] = 0;
    __syncthreads();
    const int count = sh.count;
    if (count <= kLpPool) {
      for (int i = tid; i < count; i += kThreads) {
        const LpKey k = sh.pool[i];
        int place = 0;
        for (int j = 0; j < count; ++j) place += sh.pool[j] > k;
        if (place < p.top) sh.list[place] = k;
      }
    } else {
      LpKey best_k = 0;                                        // the warp's 32 largest, lane 0 the first
      for (int i0 = warp * 32; i0 < todo; i0 += kThreads) {
        const int at = unit_of(i0 + lane);
        LpVec<T> u;
        u.raw = make_uint4(lp_shut<T>(), lp_shut<T>(), lp_shut<T>(), lp_shut<T>());
        if (at < hi) u = load_unit(at);
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float2 x = lp_pair(u, e / 2);
          const LpKey k = lp_key(e & 1 ? x.y : x.x, at * kN + e - shift), least = __shfl_sync(0xffffffffu, best_k, 31);
          if (__any_sync(0xffffffffu, k > least)) best_k = lp_merge(best_k, lp_sort(k));
        }
      }
#pragma unroll
      for (int half = kWarps / 2; half > 0; half /= 2) {
        if (warp >= half && warp < 2 * half) sh.merged[warp][lane] = best_k;
        __syncthreads();
        if (warp < half) best_k = lp_merge(best_k, sh.merged[warp + half][lane]);
      }
      if (warp == 0) sh.list[lane] = lane < p.top ? best_k : 0;
    }
    __syncthreads();
  }

  if (cluster > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");          // the first CTA runs
    uint32_t to;
    if (kTop && warp == 0) {
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(&sh.part_list[rank][lane])));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(sh.list[lane]) : "memory");
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
    mine = join(sh.part, cluster, [](const LpStats& s, float max) { return s.in_row<T>(max); });
    if constexpr (kTop) {                                      // the CTAs' lists, two by two
      for (int gap = 1; gap < cluster; gap *= 2) {
        const int c = 2 * gap * warp;
        if (c + gap < cluster) sh.part_list[c][lane] = lp_merge(sh.part_list[c][lane], sh.part_list[c + gap][lane]);
        __syncthreads();
      }
      if (tid < 32) sh.list[tid] = sh.part_list[0][tid];
      __syncthreads();
    }
  }
  const float log_s = log2f(mine.s);
  const bool bad = mine.s != mine.s, wide = lp_wide<T>(mine.m);
  auto logp = [&](float x) {
    if (bad) return nan;
    if (!(x > -INFINITY)) return -INFINITY;
    if (wide || lp_wide<T>(x)) return (x == mine.m ? 0.f : x - mine.m) - (log_s - lp_rest<T>(mine.m)) * kLpLn2;
    return (fmaf(x, kLpLog2e, -__fmul_rn(mine.m, kLpLog2e)) - log_s) * kLpLn2;
  };
  if (tid == 0) p.entropy[row] = bad ? nan : mine.s > 0.f ? (log_s - mine.w / mine.s) * kLpLn2 : 0.f;
  for (int j = tid; j < p.given; j += kThreads) {
    if (j != tid) {
      tok = token(j);
      tok_x = logit(tok);
    }
    p.logprob[row * p.given + j] = tok < 0 ? 0.f : tok >= p.vocab ? nan : logp(tok_x);
  }
  if (kTop && tid < p.top) {
    const LpKey key = bad ? 0 : sh.list[tid];
    p.top_ids[row * p.top + tid] = key ? lp_key_id(key) : -1;
    p.top_logprobs[row * p.top + tid] = bad ? nan : key ? logp(lp_key_value(key)) : -INFINITY;
  }
}

template <typename T, int kThreads, bool kLong = false>
static cudaError_t logprobs_go(const LogprobParams& p, int cluster, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.rows) * cluster), block(kThreads);
  return p.top ? launch_kernel_cluster(logprobs_kernel<T, kThreads, true, kLong>, grid, block, 0, st, cluster, 1u, p, cluster)
               : launch_kernel_cluster(logprobs_kernel<T, kThreads, false, kLong>, grid, block, 0, st, cluster, 1u, p, cluster);
}

// us a launch that decide.  Many rows: the shorter they are, the more of them an SM should have under way (2000 rows bf16 of 6000, 12000 and 50000
// with CTAs of 64, 128 and 256 threads: 8.5 / 9.7 / 13.3, 13.7 / 12.5 / 18.3, 45.5 / 40.1 / 42.6); longer rows take 128 threads only where the last wave
// of CTAs is filled as well as with 256 (700 x 50000: 25.3 and 20.0; 1500 x 32768: 24.3 and 23.4).  Few rows do not (138 x 2067 fp32 with 32
// alternatives: 9.5 with 64 threads, 6.9 with 256): a cluster shares a row, as many CTAs as the card holds at a time and no more (with 5 alternatives
// bf16: 80 x 128256 13.7 in clusters of eight with 128 threads, 16.5 with 256, which do not fit; 160 x 128256 17.0 in threes, 20.2 in fours; one row
// 7 in a cluster of eight).  Half of the places and more, in twos or alone: 300 x 32000 15.4 / 11.6, 592 x 128256 37.4 / 32.0, 500 x 128256 34.1 / 31.7;
// only 300 to 400 rows beyond 100000 logits lose by the rule (300 x 128256 27.7 / 30.5, without alternatives 22.8 / 27.5; 400 x 128256 30.1 / 31.2).
template <typename T>
static cudaError_t logprobs_go(const LogprobParams& p, cudaStream_t st) {
  const long long units = (static_cast<long long>(p.vocab) + LpVec<T>::kN - 1) / LpVec<T>::kN;
  if (units <= 256 || (units <= kLpSmallUnits && p.rows > kLpFill)) return logprobs_go<T, 64>(p, 1, st);
  if (p.rows > kLpFill && units <= 8 * kLpSmallUnits) {
    const long long of256 = (p.rows + 591LL) / 592 * 592, of128 = (p.rows + 1183LL) / 1184 * 1184;      // rows that the waves would hold
    if (units <= 2 * kLpSmallUnits || (p.rows > 1184 && of128 <= of256)) return logprobs_go<T, 128>(p, 1, st);
  }
  if (p.rows >= kLpLongRows && units >= 32 * 256) return logprobs_go<T, 256, true>(p, 1, st);
  const bool narrow = p.rows > kLpFill / kLpMaxCluster && p.rows <= 2 * kLpFill / kLpMaxCluster;
  const long long fits = units / (narrow ? 256 : 512);         // (two units a thread at least)
  const int wanted = narrow ? kLpMaxCluster : static_cast<int>(kLpFill / p.rows), cluster = static_cast<int>(std::min<long long>(std::min(wanted, kLpMaxCluster), fits));
  return narrow && cluster > 1 ? logprobs_go<T, 128>(p, cluster, st) : logprobs_go<T, 256>(p, cluster > 1 ? cluster : 1, st);
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
