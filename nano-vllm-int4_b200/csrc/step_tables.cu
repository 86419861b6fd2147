// Step metadata of a batch built on the GPU from request lengths: context
// lengths, block tables, the starts of the requests' new tokens, and the
// position and cache slot of every new token.
//
// Request b has cached[b] tokens in the cache and new[b] to compute; it owns
// the next ceil((cached + new) / page_size) entries of the flat page list.  So
// the first page of a request and its first token are two prefix sums over the
// batch, and each output element follows from them by itself.  One launch:
// every CTA makes both sums in shared memory (eight bytes a request, which limits
// the batch) and takes its share of the outputs.  3.5 us for 32 or 40
// requests, 4.6 us for 512.  Bound by latency: two loads in a row, the scan, a
// binary search.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kStepThreads = 256;

struct StepTablesArgs {
  const int* cached;
  const int* fresh;
  const int* pages;
  int* block_tables;  // [rows, max_pages]
  int* context_lens;  // [rows]
  int* query_starts;  // [rows + 1]
  int* slot_mapping;  // [tokens]
  int64_t* positions; // [tokens]
  int64_t num_listed, tokens;
  int batch, rows, max_pages, page_size;
};

// Sums are kept in 64 bits and clamped to int32 where they are stored: a
// clamped start lies beyond every output, so nothing is written for it.
__device__ __forceinline__ int clamp_i32(int64_t v) { return static_cast<int>(v < 0x7FFFFFFF ? v : 0x7FFFFFFF); }

__global__ void __launch_bounds__(kStepThreads) step_tables_kernel(const StepTablesArgs p) {
  extern __shared__ int step_smem[];
  int* page_start = step_smem;                 // [batch + 1]
  int* token_start = step_smem + p.batch + 1;  // [batch + 1]
  __shared__ int64_t warp_sums[2][kStepThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  int64_t pages_before = 0, tokens_before = 0;  // totals of the earlier rounds
  for (int b0 = 0; b0 < p.batch; b0 += kStepThreads) {
    const int b = b0 + tid;
    int64_t np = 0, nt = 0;
    if (b < p.batch) {
      nt = max(p.fresh[b], 0);
      np = (static_cast<int64_t>(max(p.cached[b], 0)) + nt + p.page_size - 1) / p.page_size;
    }
    int64_t ip = np, it = nt;  // inclusive sums
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, ip, m), c = __shfl_up_sync(0xffffffffu, it, m);
      if (lane >= m) ip += a, it += c;
    }
    if (lane == 31) warp_sums[0][warp] = ip, warp_sums[1][warp] = it;
    __syncthreads();
    int64_t bp = pages_before, bt = tokens_before;
    for (int w = 0; w < kStepThreads / 32; ++w) {
      if (w < warp) bp += warp_sums[0][w], bt += warp_sums[1][w];
      pages_before += warp_sums[0][w], tokens_before += warp_sums[1][w];
    }
    if (b < p.batch) page_start[b] = clamp_i32(bp + ip - np), token_start[b] = clamp_i32(bt + it - nt);
    __syncthreads();
  }
  if (tid == 0) page_start[p.batch] = clamp_i32(pages_before), token_start[p.batch] = clamp_i32(tokens_before);
  __syncthreads();

  const int64_t first = static_cast<int64_t>(blockIdx.x) * kStepThreads + tid;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kStepThreads;
  for (int64_t i = first; i <= p.rows; i += stride) {
    p.query_starts[i] = token_start[min(static_cast<int>(i), p.batch)];
    if (i < p.rows)
      p.context_lens[i] =
          i < p.batch ? clamp_i32(static_cast<int64_t>(max(p.cached[i], 0)) + max(p.fresh[i], 0)) : 0;
  }
  for (int64_t i = first; i < static_cast<int64_t>(p.rows) * p.max_pages; i += stride) {
    const int b = static_cast<int>(i / p.max_pages), j = static_cast<int>(i - static_cast<int64_t>(b) * p.max_pages);
    int page = 0;
    if (b < p.batch && j < page_start[b + 1] - page_start[b]) {
      const int64_t at = static_cast<int64_t>(page_start[b]) + j;
      if (at < p.num_listed) page = p.pages[at];
      else record_index_error(kErrBadPage);
    }
    p.block_tables[i] = page;
  }
  for (int64_t i = first; i < p.tokens; i += stride) {
    int slot = -1;
    int64_t position = 0;
    if (i < token_start[p.batch]) {
      int lo = 0, hi = p.batch;  // last request that starts at or before token i
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (token_start[mid] <= i) lo = mid;
        else hi = mid;
      }
      position = static_cast<int64_t>(max(p.cached[lo], 0)) + (i - token_start[lo]);
      const int64_t j = position / p.page_size, at = page_start[lo] + j;
      int64_t s = -1;
      if (j < p.max_pages && at < p.num_listed)
        s = p.pages[at] < 0 ? -1 : static_cast<int64_t>(p.pages[at]) * p.page_size + (position - j * p.page_size);
      if (s < 0 || s > 0x7FFFFFFF) record_index_error(kErrBadPage);
      else slot = static_cast<int>(s);
    }
    p.slot_mapping[i] = slot;
    p.positions[i] = position;
  }
}

int launch_step_tables(const int* cached, const int* fresh, const int* pages, int* block_tables, int* context_lens,
                       int* query_starts, int* slot_mapping, int64_t* positions, int64_t batch, int64_t rows,
                       int64_t num_listed, int64_t tokens, int64_t max_pages, int64_t page_size,
                       cudaStream_t stream) {
  StepTablesArgs a;
  a.cached = cached;
  a.fresh = fresh;
  a.pages = pages;
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.query_starts = query_starts;
  a.slot_mapping = slot_mapping;
  a.positions = positions;
  a.num_listed = num_listed;
  a.tokens = tokens;
  a.batch = static_cast<int>(batch);
  a.rows = static_cast<int>(rows);
  a.max_pages = static_cast<int>(max_pages);
  a.page_size = static_cast<int>(page_size);
  const int64_t items = std::max(std::max(rows * max_pages, tokens), rows + 1);
  const int64_t ctas = std::min<int64_t>((items + kStepThreads - 1) / kStepThreads, 2 * device_sm_count());
  static int done[64] = {};
  // For every batch: without it the static shared memory takes its part of the 48 KB.
  const int rc = ensure_smem_attr(reinterpret_cast<const void*>(&step_tables_kernel),
                                  2 * (NV4_STEP_MAX_BATCH + 1) * sizeof(int), done);
  if (rc != NV4_OK) return rc;
  const int smem = 2 * (a.batch + 1) * static_cast<int>(sizeof(int));
  return launch_kernel(step_tables_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kStepThreads),
                       smem, stream, false, a);
}

}  // namespace nv4
