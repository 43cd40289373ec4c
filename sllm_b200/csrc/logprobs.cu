// Log-probabilities of given tokens, the entropy and the largest alternatives of rows of logits:
//   m = max z,  S = sum e^(z - m),  W = sum e^(z - m) (z - m)
//   log p(t) = z_t - m - ln S,   H = -sum p ln p = ln S - W / S
// Alternatives are ordered by logit, equal ones by id.  -inf shuts a token out; a row of nothing else has log p = -inf, H = 0 and
// no alternatives (id -1).  With +inf logits the row is uniform over them; a NaN makes the row's numbers NaN and leaves no
// alternatives.  A given id below 0 stands for no token (0), one beyond the vocabulary has log p NaN.
#include <cfloat>
#include "common.cuh"
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

// Order of (logit, id) as one integer: larger logits first, then smaller ids; 0 is below every token that is not shut out.
// (x + 0 makes one value of both zeros.)
__device__ __forceinline__ unsigned long long lp_key(float x, int id) {
  const uint32_t b = __float_as_uint(x + 0.f), o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return x == -INFINITY ? 0ull : (static_cast<unsigned long long>(o) << 32) | (0x7fffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ int lp_key_id(unsigned long long k) { return static_cast<int>(0x7fffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

constexpr int kLpThreads = 256;

// One CTA per row; alternatives by one pass over the row each.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LogprobParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sf[3][kLpThreads / 32];
  __shared__ unsigned long long sk[kLpThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x;
  const T* z = static_cast<const T*>(p.logits) + row * p.ld;
  auto sum = [&](float v, int slot) {
    v = warp_sum(v);
    if (lane == 0) sf[slot][warp] = v;
    __syncthreads();
    float r = 0.f;
    for (int w = 0; w < kLpThreads / 32; ++w) r += sf[slot][w];
    return r;
  };
  float m = -FLT_MAX, bad = 0.f;
  for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
    const float x = lp_load(z + i);
    if (x != x) bad = 1.f;
    m = fmaxf(m, x);
  }
  m = warp_max(m);
  if (lane == 0) sf[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < kLpThreads / 32; ++w) m = fmaxf(m, sf[0][w]);
  bad = sum(bad, 1);
  float s = 0.f, wd = 0.f;
  for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
    const float x = lp_load(z + i);
    if (x == -INFINITY) continue;
    const float d = x == m ? 0.f : x - m, e = expf(d);
    s += e;
    if (e > 0.f) wd += e * d;
  }
  __syncthreads();
  s = sum(s, 0);
  wd = sum(wd, 2);
  const float nan = __int_as_float(0x7fffffff), ln_s = logf(s);
  auto logp = [&](float x) {
    return bad > 0.f ? nan : x == -INFINITY ? -INFINITY : (x == m ? 0.f : x - m) - ln_s;
  };
  if (threadIdx.x == 0) p.entropy[row] = bad > 0.f ? nan : s > 0.f ? ln_s - wd / s : 0.f;
  for (int j = threadIdx.x; j < p.given; j += kLpThreads) {
    const long long at = row * p.given + j;
    const long long id = p.tokens64 ? static_cast<const long long*>(p.tokens)[at] : static_cast<const int*>(p.tokens)[at];
    p.logprob[at] = id < 0 ? 0.f : id >= p.vocab ? nan : logp(lp_load(z + id));
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    if (!(bad > 0.f))
      for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
        const unsigned long long key = lp_key(lp_load(z + i), i);
        if (key < last && key > best) best = key;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long v = __shfl_xor_sync(0xffffffffu, best, o);
      best = v > best ? v : best;
    }
    __syncthreads();
    if (lane == 0) sk[warp] = best;
    __syncthreads();
    for (int w = 0; w < kLpThreads / 32; ++w) best = sk[w] > best ? sk[w] : best;
    if (threadIdx.x == 0) {
      p.top_ids[row * p.top + k] = best ? lp_key_id(best) : -1;
      p.top_logprobs[row * p.top + k] = best ? logp(lp_key_value(best)) : bad > 0.f ? nan : -INFINITY;
    }
    last = best ? best : last;
    if (!best) last = 0;
  }
}

}  // namespace sllm

using namespace sllm;

// logits [rows, vocab] of dtype 0 bf16, 1 fp16, 2 fp32, rows ld elements apart; tokens [rows, given] int32 (tokens64: int64);
// logprob [rows, given], entropy [rows], top_ids / top_logprobs [rows, top] (0 to 32, null with 0).
SLLM_EXPORT int sllm_token_logprobs(const void* logits, long long ld, int rows, int vocab, int dtype, const void* tokens, int tokens64,
                                    int given, int top, float* logprob, float* entropy, int* top_ids, float* top_logprobs, void* stream) {
  if (!logits || rows <= 0 || vocab <= 0 || ld < 0 || given < 0 || top < 0 || !entropy || dtype < 0 || dtype > 2) return SLLM_ERR_INVALID_ARGUMENT;
  if ((given && (!tokens || !logprob)) || (top && (!top_ids || !top_logprobs))) return SLLM_ERR_INVALID_ARGUMENT;
  if (top > 32) return SLLM_ERR_LIMIT;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return SLLM_ERR_ALIGNMENT;
  LogprobParams p = {logits, ld, rows, vocab, tokens, tokens64, given, top, logprob, entropy, top_ids, top_logprobs};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(rows), block(kLpThreads);
  cudaError_t e;
  if (dtype == 0) e = launch_kernel(logprobs_kernel<__nv_bfloat16>, grid, block, 0, st, 1u, p);
  else if (dtype == 1) e = launch_kernel(logprobs_kernel<__half>, grid, block, 0, st, 1u, p);
  else e = launch_kernel(logprobs_kernel<float>, grid, block, 0, st, 1u, p);
  return e == cudaSuccess ? SLLM_OK : SLLM_ERR_CUDA;
}
