// The structure of a flat batch from request lengths: request i has new[i] tokens behind starts[i] that its pages hold already, and
// its pages - ceil((starts[i] + new[i]) / page) of them - follow those of request i - 1 in one list.  With off and first the running
// sums of new and of the page counts, row r of request i is position starts[i] + r - off[i], sees position + 1 keys and is kept in
// slot pages[first[i] + position / page] * page + position % page; the table's row i holds the request's pages, then zeros.  Rows
// behind the last request: position, request and slot -1, no keys.  A request without new tokens has no last row (-1).
//
// One launch: every CTA takes the running sums of all requests into shared memory (loads out of L2, all at once) and then its share
// of the rows and of the table, so that neither a long request nor a wide table waits for one CTA.  A second launch for the sums would
// cost more than they do (2.4 us a launch at 64 requests).  Measured (us a launch, in brackets its bytes at the copy bandwidth): 64
// requests of one token 3.2 (0.03), one of 65536 tokens 3.4 (0.2), 300 with a table of 8192 columns 8.5 (2.2), 16384 requests 71 (0.3; 128 KB of
// sums hold one CTA per SM).
#include <climits>
#include "common.cuh"
#include "api.h"

namespace sllm {

struct PlanParams {
  const int *new_lens, *starts, *pages;
  int requests, rows, max_blocks, page;
  int page_count;
  long long ld_table;
  int *row_off, *positions, *seq_index, *kv_lens;
  long long *slots, *last_rows;
  int* table;
  int row_units, col_units;                 // units of rows; units of a table row
  bool vec;                                 // 16-byte stores into the table
};

constexpr int kPlanThreads = 256, kPlanRows = 512, kPlanCols = 2048, kPlanRequests = 16384, kPlanItems = 8;

// first[i] saturates: a list holds less than 2^31 pages, and what lies beyond it reads page 0.
struct __align__(8) PlanAt {
  int off, first;
  __device__ __forceinline__ PlanAt operator+(const PlanAt& o) const {
    const long long a = static_cast<long long>(off) + o.off, b = static_cast<long long>(first) + o.first;
    return {static_cast<int>(a < INT_MAX ? a : INT_MAX), static_cast<int>(b < INT_MAX ? b : INT_MAX)};
  }
};
__device__ __forceinline__ int plan_count(int start, int n, int page) {      // pages of a request
  const long long c = (static_cast<long long>(start) + n + page - 1) / page;
  return static_cast<int>(c < INT_MAX ? c : INT_MAX);
}

__global__ void __launch_bounds__(kPlanThreads) batch_plan_kernel(const PlanParams p) {
  extern __shared__ PlanAt at[];            // [requests + 1]
  __shared__ PlanAt part[kPlanThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  PlanAt carry = {0, 0};
  const int each = min((p.requests + kPlanThreads - 1) / kPlanThreads, kPlanItems);      // requests of a thread in a round, one behind the other
  for (int i0 = 0; i0 < p.requests; i0 += kPlanThreads * each) {
    const int i1 = i0 + tid * each;
    int n[kPlanItems], start[kPlanItems];
#pragma unroll
    for (int k = 0; k < kPlanItems; ++k) {
      const bool in = k < each && i1 + k < p.requests;
      n[k] = in ? p.new_lens[i1 + k] : 0;
      start[k] = in ? p.starts[i1 + k] : 0;
    }
    PlanAt own[kPlanItems], sum = {0, 0};
#pragma unroll
    for (int k = 0; k < kPlanItems; ++k) {
      const int len = max(n[k], 0);
      if (k < each && i1 + k < p.requests) sum = sum + PlanAt{len, plan_count(max(start[k], 0), len, p.page)};
      own[k] = sum;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const PlanAt u = {__shfl_up_sync(0xffffffffu, sum.off, o), __shfl_up_sync(0xffffffffu, sum.first, o)};
      if (lane >= o) sum = u + sum;
    }
    if (lane == 31) part[warp] = sum;
    const PlanAt lanes = {__shfl_up_sync(0xffffffffu, sum.off, 1), __shfl_up_sync(0xffffffffu, sum.first, 1)};
    __syncthreads();
    PlanAt before = carry;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) before = before + part[w];
      carry = carry + part[w];
    }
    if (lane) before = before + lanes;      // of all requests ahead of the thread's
#pragma unroll
    for (int k = 0; k < kPlanItems; ++k)
      if (k < each && i1 + k < p.requests) at[i1 + k + 1] = before + own[k];
    __syncthreads();
  }
  if (tid == 0) at[0] = {0, 0};
  __syncthreads();

  auto page_of = [&](int first, int c) {    // (first + c below 2^32: no wrap)
    const unsigned i = static_cast<unsigned>(first) + static_cast<unsigned>(c);
    return i < static_cast<unsigned>(p.page_count) ? p.pages[i] : 0;
  };
  const int units = p.row_units + p.requests * p.col_units;
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    if (unit < p.row_units) {
      const int end = min((unit + 1) * kPlanRows, p.rows);
      for (int r = unit * kPlanRows + tid; r < end; r += kPlanThreads) {
        if (r >= carry.off) {               // behind the last request
          p.positions[r] = p.seq_index[r] = -1;
          p.kv_lens[r] = 0;
          p.slots[r] = -1;
          continue;
        }
        int i = 0;                          // the last request that starts at or ahead of r; among equal starts the one with tokens
        for (int n = p.requests; n > 1;) {
          const int half = n >> 1;
          if (at[i + half].off <= r) i += half;
          n -= half;
        }
        const int pos = max(p.starts[i], 0) + r - at[i].off, c = pos / p.page;
        p.positions[r] = pos;
        p.seq_index[r] = i;
        p.kv_lens[r] = pos + 1;
        p.slots[r] = static_cast<long long>(page_of(at[i].first, c)) * p.page + (pos - c * p.page);
      }
    } else {
      const int u = unit - p.row_units, i = u / p.col_units, c0 = (u - i * p.col_units) * kPlanCols, end = min(c0 + kPlanCols, p.max_blocks);
      const int first = at[i].first, count = at[i + 1].first - first;
      int* row = p.table + i * p.ld_table;
      if (p.vec) {
        for (int c = c0 + tid * 4; c < end; c += kPlanThreads * 4) {
          int v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = c + k < count ? page_of(first, c + k) : 0;
          *reinterpret_cast<int4*>(row + c) = make_int4(v[0], v[1], v[2], v[3]);
        }
      } else {
        for (int c = c0 + tid; c < end; c += kPlanThreads) row[c] = c < count ? page_of(first, c) : 0;
      }
    }
  }
  if (blockIdx.x == gridDim.x - 1) {        // (the CTA with the fewest units)
    for (int i = tid; i <= p.requests; i += kPlanThreads) {
      p.row_off[i] = at[i].off;
      if (i < p.requests) p.last_rows[i] = at[i + 1].off > at[i].off ? at[i + 1].off - 1 : -1;
    }
  }
}

}  // namespace sllm

using namespace sllm;

// new_lens, starts [requests], pages [page_count]; row_off [requests + 1], positions / seq_index / kv_lens / slots [rows], last_rows
// [requests], table [requests, max_blocks] with rows ld_table apart.  Lengths below 0 count as 0; pages beyond the list read as 0
// and rows beyond `rows` are left out.  At most 16384 requests and 2^31 - 1 pages.
SLLM_EXPORT int sllm_batch_plan(const int* new_lens, const int* starts, const int* pages, long long page_count, int requests, int rows,
                                int max_blocks, long long ld_table, int page, int* row_off, int* positions, int* seq_index, int* kv_lens,
                                long long* slots, long long* last_rows, int* table, void* stream) {
  if (requests < 0 || rows < 0 || max_blocks < 0 || page <= 0 || page_count < 0 || ld_table < max_blocks) return SLLM_ERR_INVALID_ARGUMENT;
  if (!row_off || (requests && (!new_lens || !starts || !last_rows || (max_blocks && !table))) || (page_count && !pages))
    return SLLM_ERR_INVALID_ARGUMENT;
  if (rows && (!positions || !seq_index || !kv_lens || !slots)) return SLLM_ERR_INVALID_ARGUMENT;
  if (requests > kPlanRequests || page_count > INT_MAX || rows > INT_MAX - kPlanRows || max_blocks > INT_MAX - kPlanCols) return SLLM_ERR_LIMIT;
  PlanParams p = {new_lens, starts, pages, requests, rows, max_blocks, page, static_cast<int>(page_count), ld_table, row_off, positions,
                  seq_index, kv_lens, slots, last_rows, table, (rows + kPlanRows - 1) / kPlanRows, (max_blocks + kPlanCols - 1) / kPlanCols,
                  max_blocks % 4 == 0 && ld_table % 4 == 0 && (reinterpret_cast<uintptr_t>(table) & 15) == 0};
  const long long units = p.row_units + static_cast<long long>(requests) * p.col_units;
  if (units > INT_MAX) return SLLM_ERR_LIMIT;
  const size_t smem = sizeof(PlanAt) * (requests + 1);
  // (always the most that a call takes: a smaller figure would refuse the launch of a larger call on another thread; without it a launch
  // has 48 KB, the kernel's own array among them)
  constexpr int kMostSmem = static_cast<int>(sizeof(PlanAt)) * (kPlanRequests + 1);
  if (smem + sizeof(PlanAt) * (kPlanThreads / 32) > 48 * 1024 && cudaFuncSetAttribute(batch_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem) != cudaSuccess)
    return SLLM_ERR_CUDA;
  const int fill = 148 * (smem > 96 * 1024 ? 1 : smem > 48 * 1024 ? 2 : 4);
  const int ctas = static_cast<int>(units < 1 ? 1 : units < fill ? units : fill);
  return launch_kernel(batch_plan_kernel, dim3(ctas), dim3(kPlanThreads), smem, static_cast<cudaStream_t>(stream), 1u, p) == cudaSuccess
             ? SLLM_OK
             : SLLM_ERR_CUDA;
}
