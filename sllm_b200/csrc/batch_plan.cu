// The structure of a flat batch from request lengths: request i has new[i] tokens behind starts[i] that its pages hold already, and
// its pages - ceil((starts[i] + new[i]) / page) of them - follow those of request i - 1 in one list.  With off and first the running
// sums of new and of the page counts, row r of request i is position starts[i] + r - off[i], sees position + 1 keys and is kept in
// slot pages[first[i] + position / page] * page + position % page; the table's row i holds the request's pages, then zeros.  Rows
// behind the last request: position, request and slot -1, no keys.  A request without new tokens has no last row (-1).
#include "common.cuh"
#include "api.h"

namespace sllm {

struct PlanParams {
  const int *new_lens, *starts, *pages;
  int requests, rows, max_blocks, page;
  long long page_count, ld_table;
  int *row_off, *positions, *seq_index, *kv_lens;
  long long *slots, *last_rows;
  int* table;
};

constexpr int kPlanThreads = 256;

__device__ __forceinline__ int plan_new(const PlanParams& p, int i) { return max(p.new_lens[i], 0); }
__device__ __forceinline__ long long plan_pages(const PlanParams& p, int i) {
  return (static_cast<long long>(max(p.starts[i], 0)) + plan_new(p, i) + p.page - 1) / p.page;
}

// One CTA per request, one more for the rows behind the last.
__global__ void __launch_bounds__(kPlanThreads) batch_plan_kernel(const PlanParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ long long part[2][kPlanThreads / 32];
  const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long off = 0, first = 0;
  for (int j = threadIdx.x; j < i; j += kPlanThreads) {
    off += plan_new(p, j);
    first += plan_pages(p, j);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    off += __shfl_xor_sync(0xffffffffu, off, o);
    first += __shfl_xor_sync(0xffffffffu, first, o);
  }
  if (lane == 0) {
    part[0][warp] = off;
    part[1][warp] = first;
  }
  __syncthreads();
  off = first = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    off += part[0][w];
    first += part[1][w];
  }
  if (threadIdx.x == 0) p.row_off[i] = static_cast<int>(off);
  if (i == p.requests) {
    for (long long r = off + threadIdx.x; r < p.rows; r += kPlanThreads) {
      p.positions[r] = p.seq_index[r] = -1;
      p.kv_lens[r] = 0;
      p.slots[r] = -1;
    }
    return;
  }
  const int n = plan_new(p, i), start = max(p.starts[i], 0);
  const long long count = plan_pages(p, i);
  auto page_of = [&](long long c) { return first + c < p.page_count ? p.pages[first + c] : 0; };
  if (threadIdx.x == 0) p.last_rows[i] = n ? off + n - 1 : -1;
  for (int k = threadIdx.x; k < n; k += kPlanThreads) {
    const long long r = off + k;
    if (r >= p.rows) break;
    const int pos = start + k;
    p.positions[r] = pos;
    p.seq_index[r] = i;
    p.kv_lens[r] = pos + 1;
    p.slots[r] = static_cast<long long>(page_of(pos / p.page)) * p.page + pos % p.page;
  }
  int* row = p.table + static_cast<long long>(i) * p.ld_table;
  for (int c = threadIdx.x; c < p.max_blocks; c += kPlanThreads) row[c] = c < count ? page_of(c) : 0;
}

}  // namespace sllm

using namespace sllm;

// new_lens, starts [requests], pages [page_count]; row_off [requests + 1], positions / seq_index / kv_lens / slots [rows], last_rows
// [requests], table [requests, max_blocks] with rows ld_table apart.  Lengths below 0 count as 0; pages beyond the list read as 0
// and rows beyond `rows` are left out.
SLLM_EXPORT int sllm_batch_plan(const int* new_lens, const int* starts, const int* pages, long long page_count, int requests, int rows,
                                int max_blocks, long long ld_table, int page, int* row_off, int* positions, int* seq_index, int* kv_lens,
                                long long* slots, long long* last_rows, int* table, void* stream) {
  if (requests < 0 || rows < 0 || max_blocks < 0 || page <= 0 || page_count < 0 || ld_table < max_blocks) return SLLM_ERR_INVALID_ARGUMENT;
  if (!row_off || (requests && (!new_lens || !starts || !last_rows || (max_blocks && !table))) || (page_count && !pages))
    return SLLM_ERR_INVALID_ARGUMENT;
  if (rows && (!positions || !seq_index || !kv_lens || !slots)) return SLLM_ERR_INVALID_ARGUMENT;
  PlanParams p = {new_lens, starts, pages, requests, rows, max_blocks, page, page_count, ld_table, row_off, positions, seq_index, kv_lens,
                  slots, last_rows, table};
  return launch_kernel(batch_plan_kernel, dim3(requests + 1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), 1u, p) == cudaSuccess
             ? SLLM_OK
             : SLLM_ERR_CUDA;
}
