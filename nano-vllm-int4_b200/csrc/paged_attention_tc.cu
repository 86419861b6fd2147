// The two attentions of requests that share cached tokens, on the 5th-generation
// tensor cores (tcgen05 kind::f16): prompts over what their requests have cached
// (nv4_paged_prefill_attention) and the decode attention of a batch whose requests
// share a prefix (nv4_shared_prefix_attention).  BF16 cache, head_dim 128, pages of
// 256 tokens.
//
//   out = sum_t p_t v_t / sum_t p_t,   p_t = 2^(c (s_t - m)),   s_t = q . k_t,
//   c = scale * log2(e), m a running reference close to the maximum of s.
//
// Both are the same work on different rows.  A block is up to 128 rows (TB = 128 / G
// tokens with the G query heads of a KV head each) that read the same keys:
//   prompts   TB consecutive new tokens of a request (two such blocks side by side),
//             over its context up to the last one's own position;
//   prefix    up to TB requests of a group, over the pages they have in common;
//   own       one request's token, over what is left of its context.
// The keys of a block are walked in tiles of 128 (half a page).  All (block, KV head,
// tile) triples lie in one line that is cut evenly over the workers, whatever the
// lengths, so that the SMs end together; a block cut by such a border leaves
// unnormalised outputs with their references and sums, which a last kernel joins in
// the order of the tiles (the cuts follow from the lengths alone: results are
// reproducible).  A first kernel of one CTA makes the block table from the lengths on
// the device, so that captured calls follow new lengths.
//
// A CTA (one per SM, 640 threads) has two lanes: Q tile, S and O accumulators in TMEM
// (128 columns each) and two warpgroups of softmax, two threads per row.  While one
// lane's warpgroups work on its scores, the tensor cores work for the other.
//   prompts (pair)  both lanes take the same keys for two blocks of rows: K and V pass
//                   from L2 to shared memory once for 256 rows;
//   others (solo)   every lane is a worker of its own.  A decode block of up to 32 rows is
//                   spread: its rows of Q stand four times in the tile, in each quarter of
//                   the TMEM lanes, and P of quarter 2 h + t is term t of the keys of half
//                   h, zero elsewhere.  So the four schedulers share a row's exponentials,
//                   and one product does for both terms; the four parts of O are joined.
//   warp 0     copies K and V tiles (TMA, five slots of 32 KB) in the order of use
//   warps 1-2  issue S = Q K^T, O += P V of a lane each
//   warp 3     copies the lanes' rows of Q (TMA: [tokens][G heads][128 channels])
//   warps 4-19 softmax of the two lanes; outputs.  They also clear the V rows behind the last
//              token of a request (0 times an old NaN would be one)
// P goes back to TMEM over its scores.  Decode is bound by the cache's bytes: there P is
// multiplied in two BF16 terms (the upper 16 bits of the FP32 value and of the rest, 2^-14
// of it at most left out), so that the output's own rounding
// is the only one that shows (0.0017 of the norm).  Prompts are bound by the products, and
// under the power limit by their energy: there P is rounded to BF16 once (0.0023 of the
// norm; the sum of a row is that of the values before), which
// saves a third of the products.  m is moved (and O rescaled) only when a score exceeds
// it by 2^8, so O is rarely touched.  (Two tiles of queries that take turns, and the
// accumulator rescaled past a slack only, are published methods of attention for these
// tensor cores.)
//
// Measured (32 / 8 heads, the three launches): 4 prompts of 4096 tokens 656 us, 838 TFLOP/s
// (334 us at the rate of a large product); 2048 over 14,336 cached 573 us; 37 over 3100
// 22 us.  Decode of 12 groups of 8 over up to 16,384 shared tokens 135 us, 4.5 TB/s (92 us
// at the copy rate; the attention alone 111); 256 requests over 2000 168 us; 4 over 900
// 18 us, which is the three launches' latency.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kPtRows = 128;    // rows of a block, keys of a tile, head_dim
constexpr int kPtPage = 256;
constexpr int kPtMaxCtas = 160;
constexpr int kPtThreads = 640;  // a warpgroup for copies and products, two for the softmax of each lane
constexpr int kPtTile = kPtRows * kPtRows * 2;  // bytes of a Q, K or V tile
constexpr int kPtHalf = kPtTile / 2;            // 64 channels of it: [128 rows][128 bytes], 128-byte swizzle
constexpr int kPtSlots = 5;
constexpr int kPtBar = (2 + kPtSlots) * kPtTile;
constexpr int kPtTops = kPtBar + 256;           // after barriers and flags: maxima that the halves of a row exchange
constexpr int kPtSmem = kPtTops + 2 * 2 * kPtRows * 4;
constexpr float kPtSlack = 8.0f;                // log2 units by which a score may pass the reference

enum PtKind : int { kPtPrompt = 0, kPtOwn = 1, kPtPrefix = 2 };

// A block of rows and the keys it walks (for every KV head).
struct __align__(16) PtBlock {
  int seq;    // whose block table
  int tok0;   // first query token
  int ntok;   // query tokens
  int tiles;  // key tiles, at least 1
  int key0;   // first key, a multiple of the page
  int limit;  // keys that the first token sees, one more each further (prompts); the token's (own)
  int end;    // keys that exist
  int kind;
};

// Where a worker starts, and how many tiles it takes.
struct __align__(16) PtStart {
  int block, head, tile, count;
};

struct PtSums {
  int64_t total, chunk;  // cost of all blocks and heads; of a worker's share
  int blocks, prefix_blocks;
};

// The scratch: block table and borders, then the outputs of cut blocks.
struct PtScratch {
  PtSums* sums;
  PtStart* starts;   // [workers]
  PtBlock* blocks;
  int64_t* before;   // [blocks + 1]: cost (of one head) of what lies before a block
  int* row_block;    // [batch]: the prefix block of a request, or -1
  float* part;       // [workers][2][rows][128]: of a worker's first and last block, when cut
  float* part_ml;    // [..][2]: reference, sum
  float* row;        // [2][batch * Hq][4][128]: of own and prefix blocks that are not cut; four parts when spread
  float* row_ml;
};

struct PtArgs {
  const uint16_t* q;
  const int* tables;
  const int* context;
  const int* starts;  // query starts, or group starts
  const int* prefix;  // of groups, or nullptr: prompts
  uint16_t* out;
  PtScratch w;
  int64_t num_pages;
  int tokens, batch, groups, Hq, Hkv, G, TB, max_pages, workers, slot_rows;
  int block_cost;  // a block counts for its tiles and so many more, for its beginning and end
  float c;  // scale * log2(e)
};

// ------------------------------------------------------------ block table
// The block table is made by one CTA, whose time is latency (5 us, for 256 requests 7): few warps, sums of warps by
// shuffles, 32-bit divisions where they do.
constexpr int kPtPlanThreads = 512;
constexpr int kPtPlanWarps = kPtPlanThreads / 32;
constexpr int kPtPlanCached = 2048;  // blocks whose sums are kept in shared memory for the search
// Costs of all blocks below it are divided in 32 bits: in a graph 256 requests over 2000 take 151 us, 152.5 with
// divisions in 64 (4 over 900 17.3 and 17.7); what costs more takes milliseconds.
constexpr int64_t kPtNarrow = 1 << 20;

__device__ __forceinline__ int64_t pt_warp_scan(int64_t x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, m);
    if (lane >= m) x += y;
  }
  return x;
}

// Sums over the CTA of values before this thread's (two at once); `all` those of all threads.
__device__ __forceinline__ longlong2 pt_scan(int64_t v, int64_t w, int64_t (&sums)[2][kPtPlanWarps], longlong2& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t x = pt_warp_scan(v), y = pt_warp_scan(w);
  __syncthreads();
  if (lane == 31) sums[0][warp] = x, sums[1][warp] = y;
  __syncthreads();
  const int64_t a = pt_warp_scan(lane < kPtPlanWarps ? sums[0][lane] : 0);
  const int64_t b = pt_warp_scan(lane < kPtPlanWarps ? sums[1][lane] : 0);
  all.x = __shfl_sync(0xffffffffu, a, 31), all.y = __shfl_sync(0xffffffffu, b, 31);
  const int64_t u = __shfl_sync(0xffffffffu, a, max(warp - 1, 0)), t = __shfl_sync(0xffffffffu, b, max(warp - 1, 0));
  return make_longlong2((warp ? u : 0) + x - v, (warp ? t : 0) + y - w);
}

// Running maximum up to this thread, `carry` that of the threads before (updated).
__device__ __forceinline__ int pt_max_scan(int v, int (&maxima)[kPtPlanWarps], int& carry) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) x = max(x, __shfl_up_sync(0xffffffffu, x, m));
  __syncthreads();
  if (lane == 31) maxima[warp] = x;
  __syncthreads();
  const int m = lane < kPtPlanWarps ? maxima[lane] : 0;
  const int before = __reduce_max_sync(0xffffffffu, lane < warp ? m : 0);
  x = max(max(x, before), carry);
  carry = max(carry, __reduce_max_sync(0xffffffffu, m));
  return x;
}

__device__ __forceinline__ int pt_tiles(int keys) { return max(1, (keys + kPtRows - 1) / kPtRows); }
__device__ __forceinline__ int pt_cost(const PtArgs& p, int tiles) { return tiles + p.block_cost; }
// A decode block of up to 32 rows is spread: its rows stand four times in the tile.
__device__ __forceinline__ bool pt_spread(const PtArgs& p, int ntok) { return ntok <= p.TB / 4; }

__global__ void __launch_bounds__(kPtPlanThreads) pt_plan_kernel(const PtArgs p, const int block_tokens) {
  __shared__ int64_t sums[2][kPtPlanWarps];
  __shared__ int maxima[kPtPlanWarps];
  __shared__ int first[kPtPlanThreads], last[kPtPlanThreads], extra[kPtPlanThreads], which[kPtPlanThreads];
  __shared__ int table_row[kPtPlanThreads];
  __shared__ int64_t weight[kPtPlanThreads];
  __shared__ int64_t cached[kPtPlanCached];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int most = p.max_pages * kPtPage;
  grid_dependency_wait();
  grid_dependents_launch();
  int64_t tiles_before = 0;
  int blocks = 0, prefix_blocks = 0, carry = 0;
  auto put = [&](int i, int64_t before, const PtBlock& b) {
    p.w.blocks[i] = b;
    p.w.before[i] = before;
    if (i < kPtPlanCached) cached[i] = before;
  };

  if (p.prefix == nullptr) {
    for (int b0 = 0; b0 < p.batch; b0 += kPtPlanThreads) {
      const int b = b0 + tid;
      const bool live = b < p.batch;
      const int at = live ? min(max(p.starts[b], 0), p.tokens) : 0;
      const int next = live ? min(max(p.starts[b + 1], 0), p.tokens) : 0;
      const int lo = pt_max_scan(at, maxima, carry);
      first[tid] = lo;
      last[tid] = live ? max(lo, next) : lo;
      extra[tid] = live ? max(p.context[b], 0) : 0;
      __syncthreads();
      const int here = min(kPtPlanThreads, p.batch - b0);
      for (int s = warp; s < here; s += kPtPlanWarps) {
        const int n = last[s] - first[s], ctx = extra[s], end = min(ctx, most);
        int64_t sum = 0;
        for (int j = lane; j * block_tokens < n; j += 32)
          sum += pt_cost(p, pt_tiles(min(ctx - n + min(n, (j + 1) * block_tokens), end)));
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if (lane == 0) weight[s] = sum;
      }
      __syncthreads();
      const int mine = live ? (last[tid] - first[tid] + block_tokens - 1) / block_tokens : 0;
      const int64_t w = live ? weight[tid] : 0;
      longlong2 all;
      const longlong2 before = pt_scan(w, mine, sums, all);
      which[tid] = blocks + static_cast<int>(before.y);
      weight[tid] = tiles_before + before.x;
      tiles_before += all.x;
      blocks += static_cast<int>(all.y);
      __syncthreads();
      for (int s = warp; s < here; s += kPtPlanWarps) {
        const int n = last[s] - first[s], ctx = extra[s], end = min(ctx, most);
        int64_t before = weight[s];
        for (int j0 = 0; j0 * block_tokens < n; j0 += 32) {
          const int j = j0 + lane, i0 = j * block_tokens;
          const int count = min(n - i0, block_tokens);
          const int tiles = count > 0 ? pt_tiles(min(ctx - n + i0 + count, end)) : 0;
          const int cost = count > 0 ? pt_cost(p, tiles) : 0;
          const int64_t x = pt_warp_scan(cost);
          if (count > 0)
            put(which[s] + j, before + x - cost,
                PtBlock{b0 + s, first[s] + i0, count, tiles, 0, ctx - n + i0 + 1, end, kPtPrompt});
          before += __shfl_sync(0xffffffffu, x, 31);
        }
      }
      __syncthreads();
    }
  } else {
    for (int b = tid; b < p.batch; b += kPtPlanThreads) p.w.row_block[b] = -1;
    __syncthreads();
    for (int g0 = 0; g0 < p.groups; g0 += kPtPlanThreads) {
      const int g = g0 + tid;
      const bool live = g < p.groups;
      const int at = live ? min(max(p.starts[g], 0), p.batch) : 0;
      const int next = live ? min(max(p.starts[g + 1], 0), p.batch) : 0;
      const int lo = pt_max_scan(at, maxima, carry);
      first[tid] = lo;
      last[tid] = live ? max(lo, next) : lo;
      extra[tid] = live ? p.prefix[g] : 0;
      __syncthreads();
      const int here = min(kPtPlanThreads, p.groups - g0);
      for (int s = warp; s < here; s += kPtPlanWarps) {
        // the pages in common, read through the table of the longest request
        int best = 0, row = first[s], full = 0;
        for (int r = first[s] + lane; r < last[s]; r += 32) {
          const int ctx = min(p.context[r], most);
          if (ctx > best) best = ctx, row = r;
          full += ctx > 0;
        }
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) {
          const int ob = __shfl_xor_sync(0xffffffffu, best, m), orow = __shfl_xor_sync(0xffffffffu, row, m);
          if (ob > best || (ob == best && orow < row)) best = ob, row = orow;
          full += __shfl_xor_sync(0xffffffffu, full, m);
        }
        if (lane == 0) {
          extra[s] = full > 1 ? max(min(extra[s], best), 0) / kPtPage * kPtPage : 0;
          weight[s] = row;
        }
      }
      __syncthreads();
      const int shared = extra[tid], row = static_cast<int>(weight[tid]);
      const int mine = live && shared > 0 ? (last[tid] - first[tid] + p.TB - 1) / p.TB : 0;
      longlong2 all;
      const longlong2 before = pt_scan(static_cast<int64_t>(mine) * pt_cost(p, shared / kPtRows), mine, sums, all);
      which[tid] = blocks + static_cast<int>(before.y);
      weight[tid] = tiles_before + before.x;  // (the scan waited for all to have read it)
      tiles_before += all.x;
      blocks += static_cast<int>(all.y);
      table_row[tid] = row;
      __syncthreads();
      for (int s = warp; s < here; s += kPtPlanWarps) {
        if (extra[s] <= 0) continue;
        const int n = last[s] - first[s], tiles = extra[s] / kPtRows;
        for (int j = lane; j * p.TB < n; j += 32)
          put(which[s] + j, weight[s] + static_cast<int64_t>(j) * pt_cost(p, tiles),
              PtBlock{table_row[s], first[s] + j * p.TB, min(p.TB, n - j * p.TB), tiles, 0, 0, extra[s], kPtPrefix});
        for (int r = lane; r < n; r += 32) p.w.row_block[first[s] + r] = which[s] + r / p.TB;
      }
      __syncthreads();
    }
    prefix_blocks = blocks;
    for (int b0 = 0; b0 < p.batch; b0 += kPtPlanThreads) {
      const int b = b0 + tid;
      const bool live = b < p.batch;
      int tiles = 0, shared = 0, end = 0;
      if (live) {
        const int of = p.w.row_block[b];
        shared = of >= 0 ? p.w.blocks[of].end : 0;
        end = min(max(p.context[b], 0), most);
        tiles = pt_tiles(end - shared);
      }
      longlong2 all;
      const longlong2 before = pt_scan(live ? pt_cost(p, tiles) : 0, 0, sums, all);
      if (live) put(blocks + b, tiles_before + before.x, PtBlock{b, b, 1, tiles, shared, end, end, kPtOwn});
      tiles_before += all.x;
    }
    blocks += p.batch;
    __syncthreads();
  }

  const int64_t total = tiles_before * p.Hkv;
  const bool small = total < kPtNarrow;
  int64_t chunk = small ? (static_cast<uint32_t>(total) + p.workers - 1) / static_cast<uint32_t>(p.workers)
                        : (total + p.workers - 1) / p.workers;
  if (chunk < 1) chunk = 1;
  if (tid == 0) {
    p.w.before[blocks] = tiles_before;
    *p.w.sums = PtSums{total, chunk, blocks, prefix_blocks};
  }
  __syncthreads();
  const bool in_smem = blocks <= kPtPlanCached;
  // The border at `at`: block, head and tile, and the tiles (without the costs) of all before it within the block.
  auto border = [&](int64_t at, PtStart& s) {
    int lo = 0, hi = blocks - 1, cost;  // the last block that starts at or before `at`
    if (small && in_smem) {
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (static_cast<int>(cached[mid]) * p.Hkv <= static_cast<int>(at)) lo = mid;
        else hi = mid - 1;
      }
      const uint32_t into = static_cast<uint32_t>(at) - static_cast<uint32_t>(cached[lo]) * p.Hkv;
      cost = static_cast<int>((lo + 1 < blocks ? cached[lo + 1] : tiles_before) - cached[lo]);
      s.head = static_cast<int>(into / static_cast<uint32_t>(cost));
      s.tile = static_cast<int>(into % static_cast<uint32_t>(cost));
    } else {
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (p.w.before[mid] * p.Hkv <= at) lo = mid;
        else hi = mid - 1;
      }
      const int64_t into = at - p.w.before[lo] * p.Hkv;
      cost = pt_cost(p, p.w.blocks[lo].tiles);
      s.head = static_cast<int>(into / cost);
      s.tile = static_cast<int>(into % cost);
    }
    s.block = lo;
    const int tiles = cost - p.block_cost;
    // tiles before the border: what lies before it less the costs of the blocks begun (and ended) there
    const int64_t begun = static_cast<int64_t>(lo) * p.Hkv + s.head;
    const int64_t real = at - begun * p.block_cost - max(s.tile - tiles, 0);
    if (s.tile >= tiles) {  // in the block's cost: the next one begins
      s.tile = 0;
      if (++s.head == p.Hkv) s.head = 0, ++s.block;
    }
    return real;
  };
  const int64_t end = total - static_cast<int64_t>(blocks) * p.Hkv * p.block_cost;  // tiles of all
  static_assert(2 * kPtMaxCtas <= kPtPlanThreads, "a thread for every worker");
  __syncthreads();  // weight is free
  PtStart s{0, 0, 0, 0};
  const int64_t from = tid < p.workers && tid * chunk < total ? border(tid * chunk, s) : end;
  weight[tid] = from;
  __syncthreads();
  if (tid < p.workers) {
    s.count = static_cast<int>((tid + 1 < p.workers ? weight[tid + 1] : end) - from);
    p.w.starts[tid] = s;
  }
}

// ------------------------------------------------------------ tensor-core operations
// Instruction descriptor, BF16 A and B, FP32 accumulator; `b_mn`: B has its N dimension contiguous.
__host__ __device__ constexpr uint32_t pt_idesc(int m, int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Shared-memory descriptors, lower words (address and leading offset, in 16 bytes); the upper word is the same for
// both: eight rows of 128 bytes are an atom of 1024 (stride offset), 128-byte swizzle.  Q and K have their channels
// contiguous (K-major; the leading offset counts for nothing), V as the B operand its N dimension: the second 64
// channels lie a half tile on (leading offset).
constexpr uint32_t kPtDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kPtDescK = 1u << 16, kPtDescV = static_cast<uint32_t>(kPtHalf >> 4) << 16;
constexpr uint32_t kPtHalfLo = kPtHalf >> 4;
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kPtDescHi)
      : "memory");
}
// A in tensor memory
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.u32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kPtDescHi)
      : "memory");
}
__device__ __forceinline__ void pt_load_q(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ float pt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void pt_tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Registers: 640 threads are launched with 96; what the first warpgroup gives up goes to the four of the softmax, which
// hold 64 scores a thread: 64 + 4 * 104 = 5 * 96.
__device__ __forceinline__ void pt_registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 64;"); }
__device__ __forceinline__ void pt_registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 104;"); }

// Takes a lock in shared memory; after a while without it too (it only orders the lanes).
__device__ __forceinline__ void pt_lock(uint32_t* lock) {
  for (int i = 0; i < 100000; ++i)
    if (atomicCAS(lock, 0u, 1u) == 0) return;
}

__device__ __forceinline__ bool pt_passed(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// 32 bytes in one store
__device__ __forceinline__ void pt_store32(void* dst, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// The tiles of a worker, in order.  The next block's record is loaded a block ahead.
struct PtWalk {
  const PtBlock* blocks;
  PtBlock b;
  int4 ahead[2];
  int block, head, tile, heads;
  int left;    // the current one included
  bool fresh;  // the current tile is the first of this worker in its block and head

  __device__ __forceinline__ void take() {
    const int4 x = ahead[0], y = ahead[1];
    b = PtBlock{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    fetch(block + 1);
  }
  __device__ __forceinline__ void fetch(int i) {  // not the read-only path: the kernel before wrote them
    const int4* src = reinterpret_cast<const int4*>(blocks + i);
    ahead[0] = src[0], ahead[1] = src[1];
  }
  __device__ __forceinline__ void start(const PtArgs& p, int worker) {
    const PtStart s = p.w.starts[worker];
    blocks = p.w.blocks;
    block = s.block, head = s.head, tile = s.tile, heads = p.Hkv;
    left = s.count;
    fresh = true;
    if (left > 0) {
      fetch(block);
      take();
    }
  }
  // To the first tile of the next block and head.
  __device__ __forceinline__ void skip() {
    const int n = min(b.tiles - tile, left);
    tile += n - 1;
    left -= n - 1;
    next();
  }
  __device__ __forceinline__ bool last() const { return tile + 1 == b.tiles || left == 1; }  // of this worker in it
  __device__ __forceinline__ void next() {
    fresh = ++tile == b.tiles;
    --left;
    if (!fresh) return;
    tile = 0;
    if (++head == heads) {
      head = 0;
      ++block;
      if (left > 0) take();
    }
  }
};

// The same for the products, which need less of a block.
struct PtSteps {
  const PtBlock* blocks;
  int block, head, tile, heads, left, tiles, ntok, ahead_tiles, ahead_ntok;
  bool fresh;

  __device__ __forceinline__ void take() {
    tiles = ahead_tiles, ntok = ahead_ntok;
    ahead_tiles = blocks[block + 1].tiles, ahead_ntok = blocks[block + 1].ntok;
  }
  __device__ __forceinline__ void start(const PtArgs& p, int worker) {
    const PtStart s = p.w.starts[worker];
    blocks = p.w.blocks;
    block = s.block, head = s.head, tile = s.tile, heads = p.Hkv, left = s.count;
    fresh = true;
    tiles = ntok = 1;
    if (left > 0) {
      ahead_tiles = blocks[block].tiles, ahead_ntok = blocks[block].ntok;
      take();
    }
  }
  __device__ __forceinline__ bool last() const { return tile + 1 == tiles || left == 1; }
  __device__ __forceinline__ void next() {
    fresh = ++tile == tiles;
    --left;
    if (!fresh) return;
    tile = 0;
    if (++head == heads) {
      head = 0;
      ++block;
      if (left > 0) take();
    }
  }
};

struct PtBars {
  // A slot's arrival is told to the lane that it is for by a barrier of the lane's own (of a pair: one for both): on a
  // shared one a lane could take the phase before last of a slot, which the other lane has yet to see, for its own.
  uint64_t full[2][kPtSlots], empty[kPtSlots];
  uint64_t q_full[2], q_free[2], s_full[2], p_full[2], o_full[2], done;
  uint32_t tmem, lock;
  int slot_keys[kPtSlots];  // keys of the slot's tile that exist
  int lane_keys[2];         // of the tile whose scores lie in the lane
  uint32_t lane_v[2];       // its V: slot, parity of its arrival
};
static_assert(sizeof(PtBars) <= 256, "barriers");

// ------------------------------------------------------------ attention
template <bool kPair, int kTerms>
__global__ void __launch_bounds__(kPtThreads, 1)
    pt_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                        const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_q1,
                        const __grid_constant__ CUtensorMap tmap_q4, const PtArgs p) {
  extern __shared__ __align__(1024) uint8_t smem[];  // the tiles' swizzle wants multiples of 1024
  uint8_t* ring = smem + 2 * kPtTile;
  PtBars& bar = *reinterpret_cast<PtBars*>(smem + kPtBar);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPtSlots; ++s) {
      mbar_init(&bar.full[0][s], 1);
      mbar_init(&bar.full[1][s], 1);
      mbar_init(&bar.empty[s], kPair ? 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.q_full[i], 1);
      mbar_init(&bar.q_free[i], 1);
      mbar_init(&bar.s_full[i], 2);  // the products' completion, and lane_keys
      mbar_init(&bar.p_full[i], 8);  // the warps of the lane
      mbar_init(&bar.o_full[i], 1);
    }
    mbar_init(&bar.done, 2);
    bar.lock = 0;
    for (int i = 0; i < 2; ++i) bar.lane_keys[i] = 0, bar.lane_v[i] = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&bar.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // TMEM: all 512 columns are this CTA's, so they start at 0: lane l has S (then P) at l * 256, O at l * 256 + 128.
  grid_dependency_wait();  // the block table, and q, from the kernels before
  grid_dependents_launch();

  // Worker of a lane; in a pair both lanes walk worker blockIdx.x.
  auto worker = [&](int l) { return static_cast<int>(blockIdx.x) + (kPair ? 0 : l * static_cast<int>(gridDim.x)); };
  // Does lane l have rows of a block of so many tokens?  (A pair's second lane has those of the tokens behind TB.)
  auto has_rows = [&](int l, int ntok) { return !kPair || l == 0 || ntok > p.TB; };
  // Is a block of so many tokens spread (see above)?
  auto spread_out = [&](int ntok) { return kTerms == 2 && pt_spread(p, ntok); };
  // Tokens by which lane 1's rows lie further on in its tile (solo), where they fit: few rows of both lanes would
  // otherwise be the work of one of the SM's four schedulers.
  auto shift = [&](int l, int ntok) {
    return !kPair && l == 1 && !spread_out(ntok) && ntok <= p.TB / 2 ? p.TB / 2 : 0;
  };
  bool ok = true;

  if (warp < 4) pt_registers_down();
  if (warp == 0) {
    // ---------------- copies of K and V
    if (lane == 0) {
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
      uint32_t c = 0, loads[2] = {0, 0};  // ring position; bit s: parity of the lane's loads into slot s
      auto load = [&](int l, const CUtensorMap* map, int x, int row, int keys) {
        const uint32_t s = c % kPtSlots;
        uint64_t* full = &bar.full[l][s];
        if (c >= kPtSlots && !mbar_wait(&bar.empty[s], ((c / kPtSlots) - 1) & 1, kErrTimeoutEmpty)) return false;
        bar.slot_keys[s] = keys;
        mbar_arrive_expect_tx(full, keys > 0 ? kPtTile : 0);
        if (keys > 0) {
          tma_load_2d(ring + s * kPtTile, map, full, x, row);
          tma_load_2d(ring + s * kPtTile + kPtHalf, map, full, x + 64, row);
        }
        loads[l] ^= 1u << s;
        ++c;
        return true;
      };
      // the cache row and the number of keys of a walk's tile
      auto place = [&](const PtWalk& w, int& row, int& keys) {
        const int key = w.b.key0 + w.tile * kPtRows;
        row = 0;
        keys = min(max(w.b.end - key, 0), kPtRows);
        if (keys == 0) return;
        const int page = __ldg(p.tables + static_cast<int64_t>(w.b.seq) * p.max_pages + key / kPtPage);
        if (page < 0 || page >= p.num_pages) {
          record_index_error(kErrBadPage);
          keys = 0;
        } else {
          row = page * kPtPage + key % kPtPage;
        }
      };
      constexpr int kLanes = kPair ? 1 : 2;
      PtWalk w[kLanes];
      int row[kLanes], keys[kLanes], x[kLanes];
#pragma unroll
      for (int l = 0; l < kLanes; ++l) {
        w[l].start(p, worker(l));
        if (w[l].left > 0 && ok) {
          place(w[l], row[l], keys[l]);
          x[l] = w[l].head * kPtRows;
          ok = load(l, &tmap_k, x[l], row[l], keys[l]);
        }
      }
      while (ok && (w[0].left > 0 || w[kLanes - 1].left > 0)) {
#pragma unroll
        for (int l = 0; l < kLanes; ++l) {
          if (!ok || w[l].left == 0) continue;
          ok = load(l, &tmap_v, x[l], row[l], keys[l]);
          w[l].next();
          if (!ok || w[l].left == 0) continue;
          place(w[l], row[l], keys[l]);
          x[l] = w[l].head * kPtRows;
          ok = load(l, &tmap_k, x[l], row[l], keys[l]);
        }
      }
      // every copy issued must land before the CTA may exit
      for (int i = 0; i < 2 * kPtSlots; ++i) {
        const int l = i / kPtSlots, s = i % kPtSlots;
        const uint64_t start = global_timer_ns();  // (a barrier that was never used is past this parity)
        while (!mbar_try_wait(&bar.full[l][s], ((loads[l] >> s) & 1) ^ 1))
          if (global_timer_ns() - start > kWaitLimitNs) {
            record_error(kErrTimeoutDrain);
            break;
          }
      }
    }
  } else if (warp < 3) {
    // ---------------- products of a lane: S of a tile, O += P V, all by one thread.  A warp for each lane: the tensor
    // cores take few products ahead, so what one waits for in between is covered by the other's.  Of a pair's lanes one
    // at a time has its O += P V with the next S: left to themselves they fall into step, both at their exponentials
    // (the pipe of these then takes 2048 cycles) and both at their products (2048 over 14,336: 511 us in a graph, 613
    // without the lock; 4 x 4096 630 and 691, 8 ragged prompts 165 and 197).
    if (lane == 0) {
      constexpr uint32_t kQk = pt_idesc(kPtRows, kPtRows, false), kPv = pt_idesc(kPtRows, kPtRows, true);
      const uint32_t q_lo = (smem_u32(smem) >> 4) + kPtDescK, ring_lo = smem_u32(ring) >> 4;
      const int l = warp - 1;
      PtSteps w;
      w.start(p, worker(l));
      const uint32_t others = kPair ? 0 : p.w.starts[worker(1 - l)].count;
      // Ring position of V of the lane's tile i; K of the next is the one behind it.  Solo: both lanes' first K, then
      // in turn V of a tile and K of the next, while a lane has any.
      auto v_position = [&](uint32_t i) -> uint32_t {
        if (kPair) return 2 * i + 1;
        const uint32_t j = i + l;  // turns that the other lane had
        return 1 + 2 * i + (others > 0 ? 1 + min(j, others) + min(j, others - 1) : 0);
      };
      auto arrived = [&](uint64_t& b, uint32_t phase) { return mbar_wait(&b, phase & 1, kErrTimeoutMma); };
      uint32_t parts = 0, seen = 0;  // blocks so far; bit s: parity of what this lane has had in slot s
      auto filled = [&](uint32_t s) {
        const uint32_t phase = seen >> s;
        seen ^= 1u << s;
        return arrived(bar.full[kPair ? 0 : l][s], phase);
      };
      // K of the walk's tile, in slot s, and with a block's first tile its rows of Q
      auto ready = [&](uint32_t s, bool rows) {
        return filled(s) && (!rows || !w.fresh || arrived(bar.q_full[l], parts++));
      };
      // S = Q K^T
      auto scores = [&](uint32_t i, uint32_t s, bool rows) {
        if (!rows) {
          mbar_arrive(&bar.empty[s]);
          return;
        }
        tc_fence_after();
        bar.lane_keys[l] = bar.slot_keys[s];  // before the slot can be released
        const uint32_t vs = v_position(i) % kPtSlots;
        bar.lane_v[l] = vs << 1 | ((seen >> vs) & 1);
        const uint32_t qa = q_lo + l * (kPtTile >> 4), ka = ring_lo + s * (kPtTile >> 4) + kPtDescK;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t off = (j >> 2) * kPtHalfLo + (j & 3) * 2;
          pt_mma_ss(l * 256, qa + off, ka + off, kQk, j > 0);
        }
        umma_commit(&bar.s_full[l]);
        mbar_arrive(&bar.s_full[l]);
        umma_commit(&bar.empty[s]);
        if (w.last()) umma_commit(&bar.q_free[l]);
      };
      bool rows = has_rows(l, w.ntok), started = false;  // started: O holds something of the current block
      uint32_t tiles = 0;                                // with rows, so far
      uint32_t c = !kPair && l == 1 && others > 0;       // ring position
      if (w.left > 0) {
        ok = ready(c % kPtSlots, rows);
        if (ok) scores(0, c % kPtSlots, rows);
      }
      for (uint32_t i = 0; ok && w.left > 0; ++i) {
        // what O += P V and the next S need besides P
        c = v_position(i);
        const uint32_t s = c % kPtSlots, next = (c + 1) % kPtSlots;
        const bool fresh = w.fresh, last = w.last(), now = rows, spread = spread_out(w.ntok);
        if (!filled(s)) break;
        w.next();
        rows = has_rows(l, w.ntok);
        // (solo: K may be on its way from memory, and the slot of V is wanted)
        if (kPair && w.left > 0 && !ready(next, rows)) break;
        if (now) {
          const int keys = bar.slot_keys[s], steps = (keys + 15) / 16;
          if (fresh) started = false;
          const uint32_t va = ring_lo + s * (kPtTile >> 4) + kPtDescV, o = l * 256 + 128;
          // 16 keys: P, or its two terms against the same rows of V
          auto step = [&](int k, uint32_t accumulate) {
            if (kTerms == 1 || spread) {
              pt_mma_ts(o, l * 256 + (k >> 2) * 64 + (k & 3) * 8, va + k * 128, kPv, accumulate);
            } else {
              const uint32_t pk = l * 256 + (k >> 1) * 32 + (k & 1) * 8;
              pt_mma_ts(o, pk, va + k * 128, kPv, accumulate);
              pt_mma_ts(o, pk + 16, va + k * 128, kPv, 1);
            }
          };
          if (!arrived(bar.p_full[l], tiles++)) break;
          if (kPair) pt_lock(&bar.lock);
          tc_fence_after();
          if (steps == 8) {
            step(0, started);
#pragma unroll
            for (int k = 1; k < 8; ++k) step(k, 1);
          } else {
            for (int k = 0; k < steps; ++k) step(k, started || k > 0);
          }
          umma_commit(&bar.empty[s]);
          if (last) umma_commit(&bar.o_full[l]);
          started = started || steps > 0;
        } else {
          mbar_arrive(&bar.empty[s]);
        }
        if (!kPair && w.left > 0 && !ready(next, rows)) break;
        if (w.left > 0) scores(i + 1, next, rows);
        if (kPair && now) atomicExch(&bar.lock, 0u);
      }
      umma_commit(&bar.done);  // all issued products must finish before the TMEM is released
      const uint64_t start = global_timer_ns();
      while (!mbar_try_wait(&bar.done, 0))
        if (global_timer_ns() - start > kWaitLimitNs) {
          record_error(kErrTimeoutDrain);
          break;
        }
    }
    __syncwarp();
  } else if (warp < 4) {
    // ---------------- rows of Q of both lanes, by one thread.  The box takes as many tokens as a block can have; rows
    // behind the block's last (and, with a shift, before its first) are never used.
    if (lane == 0) {
      PtWalk w[2];
      int copied[2] = {0, 0};
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        w[l].start(p, worker(l));
        while (w[l].left > 0 && !has_rows(l, w[l].b.ntok)) w[l].skip();
      }
      uint64_t start = global_timer_ns();
      while (w[0].left > 0 || w[1].left > 0) {
        bool any = false;
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          if (w[l].left <= 0 || (copied[l] > 0 && !pt_passed(&bar.q_free[l], (copied[l] - 1) & 1))) continue;
          const bool one = w[l].b.kind == kPtOwn, spread = spread_out(w[l].b.ntok);
          const CUtensorMap* map = one ? &tmap_q1 : spread ? &tmap_q4 : &tmap_q;
          const int copies = spread ? 4 : 1;  // (an own block is spread: one token, up to 16 rows)
          const int token = w[l].b.tok0 + (kPair ? l * p.TB : 0) - shift(l, w[l].b.ntok);
          uint8_t* dst = smem + l * kPtTile;
          mbar_arrive_expect_tx(&bar.q_full[l], copies * (one ? 1 : spread ? p.TB / 4 : p.TB) * p.G * kPtRows * 2);
          for (int i = 0; i < copies; ++i, dst += 32 * 128) {
            pt_load_q(dst, map, &bar.q_full[l], 0, w[l].head * p.G, token);
            pt_load_q(dst + kPtHalf, map, &bar.q_full[l], 64, w[l].head * p.G, token);
          }
          ++copied[l];
          do w[l].skip();
          while (w[l].left > 0 && !has_rows(l, w[l].b.ntok));
          any = true;
        }
        if (any) {
          start = global_timer_ns();
        } else {
          __nanosleep(20);
          if (error_raised()) break;
          if (global_timer_ns() - start > kWaitLimitNs) {
            record_error(kErrTimeoutEmpty);
            break;
          }
        }
      }
#pragma unroll
      for (int l = 0; l < 2; ++l) {  // the last copies must land before the CTA may exit
        start = global_timer_ns();
        while (copied[l] > 0 && !mbar_try_wait(&bar.q_full[l], (copied[l] - 1) & 1))
          if (global_timer_ns() - start > kWaitLimitNs) {
            record_error(kErrTimeoutDrain);
            break;
          }
      }
    }
  } else {
    // ---------------- softmax and outputs: two threads a row (head r % G of its lane's token r / G), each with half of
    // a tile's keys, and of the output's channels at the end.  (With one thread a row the two warps of a scheduler left
    // two thirds of its issue slots empty.)
    pt_registers_up();
    const int l = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t at = l * 256 + half * 64 + (static_cast<uint32_t>(quarter * 32) << 16);
    float* const tops = reinterpret_cast<float*>(smem + kPtTops) + l * 2 * kPtRows;
    // Spread, a row is the work of four warps, one in each quarter: of quarter 2 h + t those of half h, for term t.
    const bool works = half == quarter >> 1;
    bool spread = false;
    float *mine = nullptr, *others = nullptr;  // the maxima of the two halves of a row
    int pairing = 0, paired = 0;               // named barrier of the warps that share rows, and its threads
    const float c = p.c;
    PtWalk w;
    w.start(p, worker(l));
    int tile = 0, part = 0, row_in = 0, limit = 0, token = 0, head = 0, from = 0;
    bool live = false, started = false;
    float m = -INFINITY, sum = 0.0f;
    // A wait that gave up does not end the walk (the warps of a row meet at barriers): later ones are not waited for.
    // From there on lane_keys may be of another tile, and differ between the warps of a row: which barriers a warp
    // meets follows from the walk alone, and V is touched by warps whose waits all ended well.
    for (; w.left > 0; w.next()) {
      if (!has_rows(l, w.b.ntok)) continue;
      if (w.fresh) {
        spread = spread_out(w.b.ntok);
        row_in = spread ? lane : r - shift(l, w.b.ntok) * p.G;
        mine = tops + half * kPtRows + (spread ? lane : r), others = tops + (1 - half) * kPtRows + (spread ? lane : r);
        pairing = spread ? 9 + l : 1 + l * 4 + quarter, paired = spread ? 128 : 64;
        const int t0 = kPair ? l * p.TB : 0, t = max(row_in, 0) / p.G;
        live = row_in >= 0 && row_in < min(w.b.ntok - t0, p.TB) * p.G;
        token = w.b.tok0 + t0 + t;
        head = w.head * p.G + row_in - t * p.G;
        limit = 0;
        if (live)
          limit = w.b.kind == kPtPrompt ? w.b.limit + t0 + t
                  : w.b.kind == kPtOwn  ? w.b.limit
                                        : __ldg(p.context + token);
        m = -INFINITY, sum = 0.0f;
        started = false;
        from = w.tile;
      }
      const bool busy = __any_sync(0xffffffffu, live);
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar.s_full[l], tile & 1, kErrTimeoutMma));
      tc_fence_after();
      const int keys = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&bar.lane_keys[l]), 0);
      if (spread && !works) {  // keys that are not this quarter's
        if (keys > 0) {
          uint32_t zero[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) zero[i] = 0u;
          pt_tmem_st16(at, zero);
          pt_tmem_st16(at + 16, zero);
          tmem_wait_st();
        }
      } else if (busy && keys <= 0) {  // no page, or a request without tokens
        named_barrier_sync(pairing, paired);
      } else if (busy) {
        const int seen = min(max(limit - (w.b.key0 + w.tile * kPtRows), 0), keys);
        const bool edge = __any_sync(0xffffffffu, live && seen < kPtRows);  // other rows may come to anything
        uint32_t s[64];
        tmem_ld32(at, s);
        tmem_ld32(at + 32, s + 32);
        tmem_wait_ld();
        if (edge) {  // what the row does not see
          const int here = seen - 64 * half;
#pragma unroll
          for (int j = 0; j < 64; ++j) s[j] = j < here ? s[j] : 0xFF800000u;
        }
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 64; j += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            t[i] = fmaxf(t[i], fmaxf(__uint_as_float(s[j + 2 * i]), __uint_as_float(s[j + 2 * i + 1])));
        float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        *mine = top;  // (spread, two warps write the same)
        named_barrier_sync(pairing, paired);
        top = fmaxf(top, *others);
        const bool move = live && top > m && (m == -INFINITY || (top - m) * c > kPtSlack);
        if (__any_sync(0xffffffffu, move) && started) {
          const float f = move ? pt_exp2((m - top) * c) : 1.0f;
          sum *= f;
#pragma unroll 1
          for (int i = 0; i < (spread ? 8 : 4); ++i) {  // half of the row's channels, or all
            const uint32_t ao = (spread ? at - half * 64 : at) + 128 + 16 * i;
            uint32_t o[16];
            tmem_ld16(ao, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            pt_tmem_st16(ao, o);
          }
        }
        if (move) m = top;
        const float base = m == -INFINITY ? 0.0f : m;
        const uint64_t base2 = pair(base, base), c2 = pair(c, c);
        uint64_t sums[2] = {0, 0};
        // The probabilities take columns of their scores: of 32 keys 16, or 16 of the upper and 16 of the lower terms
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x, y;
            const int k = 32 * i + 2 * j;
            unpair(mul2(sub2(pair(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), base2), c2), x, y);
            x = pt_exp2(x), y = pt_exp2(y);
            const uint64_t e = pair(x, y);
            sums[j & 1] = add2(sums[j & 1], e);
            if constexpr (kTerms == 1) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
              hi[j] = *reinterpret_cast<const uint32_t*>(&b);
            } else {
              const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
              hi[j] = __byte_perm(xb, yb, 0x7632);
              float u, w;
              unpair(sub2(e, pair(__uint_as_float(xb & 0xFFFF0000u), __uint_as_float(yb & 0xFFFF0000u))), u, w);
              lo[j] = __byte_perm(__float_as_uint(u), __float_as_uint(w), 0x7632);
            }
          }
          if (kTerms == 1) {
            pt_tmem_st16(at + 16 * i, hi);
          } else if (!spread) {
            pt_tmem_st16(at + 32 * i, hi);
            pt_tmem_st16(at + 32 * i + 16, lo);
          } else if (quarter & 1) {
            pt_tmem_st16(at + 16 * i, lo);
          } else {
            pt_tmem_st16(at + 16 * i, hi);
          }
        }
        float x, y;
        unpair(add2(sums[0], sums[1]), x, y);
        sum += x + y;
        tmem_wait_st();
      }
      started = started || keys > 0;
      if (keys & 15) {  // V rows behind the last key are cleared: P is zero there, they may be anything
        const uint32_t v = *reinterpret_cast<volatile uint32_t*>(&bar.lane_v[l]);
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar.full[kPair ? 0 : l][v >> 1], v & 1, kErrTimeoutFull));
        const int e = (half * 4 + quarter) * 32 + lane, row = keys + (e >> 4);
        if (ok && row < ((keys + 15) & ~15))
          *reinterpret_cast<uint4*>(ring + (v >> 1) * kPtTile + (e & 8 ? kPtHalf : 0) + row * 128 + (e & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full[l]);
      ++tile;
      if (!w.last()) continue;

      // the block's end, or this worker's: outputs
      const bool whole = from == 0 && w.tile + 1 == w.b.tiles;
      const bool final_ = kTerms == 1 && whole;
      // BF16 rows; or FP32 ones for the joining kernel, of a block that is not cut row after row, of a cut one with the
      // rows beside each other, 16 bytes each, so that a warp's stores are contiguous
      const int64_t row = static_cast<int64_t>(token) * p.Hq + head;
      uint4* dst;
      int64_t stride = 1;
      float2* ml = nullptr;
      float f = 1.0f;
      if (busy) {
        if (!spread) {
          named_barrier_sync(pairing, paired);  // the last tile's maxima are read
          *mine = sum;
          named_barrier_sync(pairing, paired);
          const float other = *others;
          named_barrier_sync(pairing, paired);
          sum = half == 0 ? sum + other : other + sum;
        }
        if (final_) {
          f = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
          dst = reinterpret_cast<uint4*>(p.out + row * kPtRows) + half * 8;
        } else if (whole) {
          const int64_t i =
              ((w.b.kind == kPtPrefix ? static_cast<int64_t>(p.batch) * p.Hq : 0) + row) * 4 + (spread ? quarter : 0);
          dst = reinterpret_cast<uint4*>(p.w.row) + i * 32 + half * 16;
          ml = reinterpret_cast<float2*>(p.w.row_ml) + i;
        } else {
          const int64_t slot = (static_cast<int64_t>(worker(l)) * 2 + (from == 0)) * (kPair ? 2 : 1) + (kPair ? l : 0);
          stride = p.slot_rows;
          const int at_row = spread ? r : row_in;
          dst = reinterpret_cast<uint4*>(p.w.part) + (slot * 32 + half * 16) * stride + at_row;
          ml = reinterpret_cast<float2*>(p.w.part_ml) + slot * stride + at_row;
        }
      }
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar.o_full[l], part & 1, kErrTimeoutMma));
      ++part;
      tc_fence_after();
      if (busy) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          uint32_t o[16];
          if (started) {
            tmem_ld16(at + 128 + 16 * i, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = 0u;
          }
          if (live && final_) {
            uint32_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const __nv_bfloat162 b =
                  __floats2bfloat162_rn(__uint_as_float(o[2 * j]) * f, __uint_as_float(o[2 * j + 1]) * f);
              v[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
            pt_store32(dst, v);
            dst += 2;
          } else if (live) {
#pragma unroll
            for (int j = 0; j < 4; ++j, dst += stride)
              *dst = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
          __syncwarp();
        }
        if (live && !final_ && (spread ? works : half == 0)) *ml = make_float2(m, spread && (quarter & 1) ? 0.0f : sum);
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(bar.tmem, 512);
  }
}

// ------------------------------------------------------------ joining
// out = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(c (m_i - max m)), in the order of the pieces.  A CTA of 128 threads
// takes four rows at a time: thread = four channels (threadIdx / 4) of a row (threadIdx % 4), so that the pieces of a
// cut block, which have the rows beside each other, are read in whole sectors.
struct PtJoin {
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

  __device__ __forceinline__ void fold(const float2& ml, const float4& v, float c) {
    const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.0f : top;
    const float a = pt_exp2((m - base) * c), b = pt_exp2((ml.x - base) * c);
    l = l * a + ml.y * b;
    o.x = o.x * a + v.x * b, o.y = o.y * a + v.y * b, o.z = o.z * a + v.z * b, o.w = o.w * a + v.w * b;
    m = top;
  }
  // Pieces `first` .. `last` of a cut block: slot 1 of the first worker, 0 of the others; `of_pair` which of a pair's.
  // kParts parts of each (of a spread row, 32 rows apart); kAhead loads in flight.
  template <int kPer, int kParts, int kAhead>
  __device__ __forceinline__ void pieces(const PtArgs& p, int first, int last, int of_pair, int row, int j) {
    for (int w0 = first; w0 <= last; w0 += kAhead / kParts) {
      float2 ml[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int w = w0 + i / kParts, at = row + 32 * (i % kParts);
        if (w > last) break;
        const int64_t slot = (static_cast<int64_t>(w) * 2 + (w == first)) * kPer + of_pair;
        ml[i] = *reinterpret_cast<const float2*>(p.w.part_ml + (slot * p.slot_rows + at) * 2);
        v[i] = *(reinterpret_cast<const float4*>(p.w.part) + (slot * 32 + j) * p.slot_rows + at);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (w0 + i / kParts <= last) fold(ml[i], v[i], p.c);
    }
  }
  // kParts parts of a row of a block that is not cut.
  template <int kParts>
  __device__ __forceinline__ void uncut(const PtArgs& p, int64_t at, int j) {
    float2 ml[kParts];
    float4 v[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      ml[i] = *reinterpret_cast<const float2*>(p.w.row_ml + (at + i) * 2);
      v[i] = *(reinterpret_cast<const float4*>(p.w.row + (at + i) * kPtRows) + j);
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) fold(ml[i], v[i], p.c);
  }
  __device__ __forceinline__ void store(uint16_t* row, int j) const {
    const float f = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * f, o.y * f), y = __floats2bfloat162_rn(o.z * f, o.w * f);
    *(reinterpret_cast<uint2*>(row) + j) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
};

constexpr int kPtJoinSplit = 32;  // CTAs that share the rows of a cut block

// Prompts: CTA (i, y) joins the block that worker i + 1 starts within, when it began in worker i.
template <bool kPair>
__global__ void __launch_bounds__(128) pt_join_prompts_kernel(const PtArgs p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const int i = blockIdx.x + 1, j = threadIdx.x >> 2;
  const PtStart s = p.w.starts[i];
  const int64_t chunk = p.w.sums->chunk;
  if (s.tile == 0 || s.tile > chunk) return;
  const PtBlock b = p.w.blocks[s.block];
  const int last = i - 1 + static_cast<int>((chunk - s.tile + b.tiles - 1) / chunk);  // with the last tile
  const int per = p.TB * p.G;  // rows of a lane
  for (int r = blockIdx.y * 4 + (threadIdx.x & 3); r < b.ntok * p.G; r += 4 * kPtJoinSplit) {
    const int l = kPair && r >= per;
    PtJoin join;
    join.pieces<kPair ? 2 : 1, 1, 8>(p, i - 1, last, l, r - l * per, j);
    const int t = r / p.G;
    join.store(p.out + (static_cast<int64_t>(b.tok0 + t) * p.Hq + s.head * p.G + r - t * p.G) * kPtRows, j);
  }
}

// Decode: CTA (request, KV head) joins what the request's own block and its group's left.  `kWide`: 128 threads as
// above for each of the four parts of spread rows (a row that is not spread is all in the first), which are joined
// last: 4 requests over 900 tokens 18 us instead of 21.  With more CTAs than fit at once the other way (256 requests:
// 184 us instead of 190).
template <bool kWide>
__global__ void __launch_bounds__(kWide ? 512 : 128, kWide ? 2 : 4) pt_join_decode_kernel(const PtArgs p) {
  __shared__ float parts[kWide ? 3 : 1][6][128];
  grid_dependency_wait();
  grid_dependents_launch();
  const int b = blockIdx.x, h = blockIdx.y, part = threadIdx.x >> 7, in_part = threadIdx.x & 127, j = in_part >> 2;
  const PtSums sums = *p.w.sums;
  const int of = p.w.row_block[b];
  const int own = sums.prefix_blocks + b;
  // the workers of a block: first and last
  auto workers = [&](int64_t before, int tiles, int& first, int& last) {
    const int64_t at = before * p.Hkv + static_cast<int64_t>(h) * pt_cost(p, tiles);
    if (sums.total < kPtNarrow) {
      const uint32_t chunk = static_cast<uint32_t>(sums.chunk), a = static_cast<uint32_t>(at);
      first = static_cast<int>(a / chunk);
      last = static_cast<int>((a + tiles - 1) / chunk);
    } else {
      first = static_cast<int>(at / sums.chunk);
      last = static_cast<int>((at + tiles - 1) / sums.chunk);
    }
  };
  int own_first, own_last, common_first = 0, common_last = 0;
  workers(p.w.before[own], p.w.blocks[own].tiles, own_first, own_last);
  int common_row = 0;
  bool common_spread = false;
  if (of >= 0) {
    const PtBlock common = p.w.blocks[of];
    workers(p.w.before[of], common.tiles, common_first, common_last);
    common_row = b - common.tok0;
    common_spread = pt_spread(p, common.ntok);
  }
  for (int g0 = 0; g0 < p.G; g0 += 4) {
    const int g = min(g0 + (in_part & 3), p.G - 1);
    PtJoin join;
    const int64_t row = static_cast<int64_t>(b) * p.Hq + h * p.G + g;
    auto add = [&](int first, int last, int in, int64_t area, bool spread) {
      if (part > 0 && !spread) return;
      const int64_t at = (area * p.batch * p.Hq + row) * 4 + part;
      if (kWide || !spread) {
        if (first < last) join.pieces<1, 1, 4>(p, first, last, 0, in + 32 * part, j);
        else join.uncut<1>(p, at, j);
      } else {
        if (first < last) join.pieces<1, 4, 4>(p, first, last, 0, in, j);
        else join.uncut<4>(p, at, j);
      }
    };
#pragma unroll 1
    for (int i = of >= 0 ? 0 : 1; i < 2; ++i)  // in one copy of the code: registers
      add(i ? own_first : common_first, i ? own_last : common_last, i ? g : common_row * p.G + g, 1 - i,
          i ? pt_spread(p, 1) : common_spread);
    if constexpr (kWide) {
      __syncthreads();
      if (part > 0) {
        const float v[6] = {join.m, join.l, join.o.x, join.o.y, join.o.z, join.o.w};
#pragma unroll
        for (int i = 0; i < 6; ++i) parts[part - 1][i][in_part] = v[i];
      }
      __syncthreads();
      if (part > 0) continue;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const auto v = [&](int k) { return parts[i][k][in_part]; };
        join.fold(make_float2(v(0), v(1)), make_float4(v(2), v(3), v(4), v(5)), p.c);
      }
    }
    if (g == g0 + (in_part & 3)) join.store(p.out + row * kPtRows, j);
  }
}

// ------------------------------------------------------------ host side
struct PtLayout {
  PtScratch w;
  int64_t bytes;
};

// `blocks` an upper bound; `rows` of a slot; `joined` rows of the decode's uncut blocks.
static PtLayout pt_layout(char* base, int64_t blocks, int64_t batch, int64_t rows, int64_t joined) {
  PtLayout l;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* q = base + at;
    at += (bytes + 255) / 256 * 256;
    return q;
  };
  constexpr int64_t kWorkers = 2 * kPtMaxCtas;
  l.w.sums = reinterpret_cast<PtSums*>(take(sizeof(PtSums)));
  l.w.starts = reinterpret_cast<PtStart*>(take(kWorkers * sizeof(PtStart)));
  l.w.blocks = reinterpret_cast<PtBlock*>(take((blocks + 1) * sizeof(PtBlock)));  // the walks load one ahead
  l.w.before = reinterpret_cast<int64_t*>(take((blocks + 1) * 8));
  l.w.row_block = reinterpret_cast<int*>(take(joined ? batch * 4 : 0));
  l.w.part = reinterpret_cast<float*>(take(kWorkers * 2 * rows * kPtRows * 4));
  l.w.part_ml = reinterpret_cast<float*>(take(kWorkers * 2 * rows * 8));
  l.w.row = reinterpret_cast<float*>(take(joined * kPtRows * 4));
  l.w.row_ml = reinterpret_cast<float*>(take(joined * 8));
  l.bytes = at;
  return l;
}

static int64_t pt_slot_rows(int64_t tokens, int64_t group) {
  return std::min<int64_t>(tokens, kPtRows / group) * group;
}

static PtLayout pt_prefill_layout(char* base, int64_t tokens, int64_t batch, int64_t num_heads, int64_t num_kv_heads) {
  const int64_t group = num_heads / num_kv_heads;
  return pt_layout(base, tokens / (kPtRows / group) + batch, batch, pt_slot_rows(tokens, group), 0);
}

static PtLayout pt_shared_layout(char* base, int64_t batch, int64_t groups, int64_t num_heads, int64_t num_kv_heads) {
  const int64_t group = num_heads / num_kv_heads;
  return pt_layout(base, batch / (kPtRows / group) + groups + batch, batch, kPtRows, 8 * batch * num_heads);
}

int64_t paged_prefill_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t num_heads,
                                                int64_t num_kv_heads) {
  return pt_prefill_layout(nullptr, tokens, batch, num_heads, num_kv_heads).bytes;
}

int64_t shared_prefix_attention_workspace_bytes(int64_t batch, int64_t groups, int64_t num_heads,
                                                int64_t num_kv_heads) {
  return pt_shared_layout(nullptr, batch, groups, num_heads, num_kv_heads).bytes;
}

template <bool kPair, int kTerms>
static int launch_pt(PtArgs& a, const void* k_cache, const void* v_cache, cudaStream_t stream) {
  static int done[64] = {};
  auto* kern = &pt_attention_kernel<kPair, kTerms>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kPtSmem, done);
  if (rc != NV4_OK) return rc;
  const int sms = std::min(device_sm_count(), kPtMaxCtas);
  if (sms <= 0) return NV4_ERR_CUDA;
  CUtensorMap maps[5] = {};
  const uint64_t rows = static_cast<uint64_t>(a.num_pages) * kPtPage, cols = static_cast<uint64_t>(a.Hkv) * kPtRows;
  if (!make_tensor_map_2d(&maps[0], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, k_cache, rows, cols, kPtRows, 64,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&maps[1], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, v_cache, rows, cols, kPtRows, 64,
                          CU_TENSOR_MAP_SWIZZLE_128B))
    return NV4_ERR_CUDA;
  // q as [tokens][heads][128]: as many tokens as a block has, one, or those of a spread block
  const uint64_t q_dims[3] = {kPtRows, static_cast<uint64_t>(a.Hq), static_cast<uint64_t>(a.tokens)};
  const uint64_t q_strides[2] = {kPtRows * 2, static_cast<uint64_t>(a.Hq) * kPtRows * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(a.G), static_cast<uint32_t>(a.TB)};
  const uint32_t box1[3] = {64, static_cast<uint32_t>(a.G), 1};
  const uint32_t box4[3] = {64, static_cast<uint32_t>(a.G), static_cast<uint32_t>(a.TB / 4)};
  if (!make_tensor_map_3d(&maps[2], CU_TENSOR_MAP_DATA_TYPE_UINT16, a.q, q_dims, q_strides, box,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_3d(&maps[3], CU_TENSOR_MAP_DATA_TYPE_UINT16, a.q, q_dims, q_strides, box1,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_3d(&maps[4], CU_TENSOR_MAP_DATA_TYPE_UINT16, a.q, q_dims, q_strides, box4,
                          CU_TENSOR_MAP_SWIZZLE_128B))
    return NV4_ERR_CUDA;
  a.workers = kPair ? sms : 2 * sms;
  rc = launch_kernel(pt_plan_kernel, dim3(1), dim3(kPtPlanThreads), 0, stream, true, a, kPair ? 2 * a.TB : a.TB);
  if (rc != NV4_OK) return rc;
  rc = launch_kernel(kern, dim3(sms), dim3(kPtThreads), kPtSmem, stream, true, maps[0], maps[1], maps[2], maps[3],
                     maps[4], a);
  if (rc != NV4_OK) return rc;
  if (a.prefix == nullptr)
    return launch_kernel(pt_join_prompts_kernel<kPair>, dim3(a.workers - 1, kPtJoinSplit), dim3(128), 0, stream, true,
                         a);
  if (static_cast<int64_t>(a.batch) * a.Hkv <= 2 * sms)
    return launch_kernel(pt_join_decode_kernel<true>, dim3(a.batch, a.Hkv), dim3(512), 0, stream, true, a);
  return launch_kernel(pt_join_decode_kernel<false>, dim3(a.batch, a.Hkv), dim3(128), 0, stream, true, a);
}

static PtArgs pt_args(const void* q, const int* block_tables, const int* context_lens, const int* starts,
                      const int* prefix, void* out, const PtScratch& w, int64_t tokens, int64_t batch, int64_t groups,
                      int64_t num_heads, int64_t num_kv_heads, int64_t num_pages, int64_t max_pages, float scale) {
  PtArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.tables = block_tables;
  a.context = context_lens;
  a.starts = starts;
  a.prefix = prefix;
  a.out = static_cast<uint16_t*>(out);
  a.w = w;
  a.num_pages = num_pages;
  a.tokens = static_cast<int>(tokens);
  a.batch = static_cast<int>(batch);
  a.groups = static_cast<int>(groups);
  a.Hq = static_cast<int>(num_heads);
  a.Hkv = static_cast<int>(num_kv_heads);
  a.G = a.Hq / a.Hkv;
  a.TB = kPtRows / a.G;
  a.max_pages = static_cast<int>(max_pages);
  a.workers = 0;
  // Prompts' blocks (4 x 4096: 662 us, 730 with none and 665 with two); a decode block's beginning is covered by the
  // other lane's products (256 over 2k: 174 us, 181 with one and 186 with two).
  a.block_cost = prefix ? 0 : 1;
  a.slot_rows = static_cast<int>(prefix ? kPtRows : pt_slot_rows(tokens, a.G));
  a.c = scale * 1.4426950408889634f;
  return a;
}

int launch_paged_prefill_attention(const void* q, const void* k_cache, const void* v_cache, const int* block_tables,
                                   const int* context_lens, const int* query_starts, void* out, void* workspace,
                                   int64_t tokens, int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                   int64_t num_pages, int64_t max_pages, float scale, cudaStream_t stream) {
  const PtLayout l = pt_prefill_layout(static_cast<char*>(workspace), tokens, batch, num_heads, num_kv_heads);
  PtArgs a = pt_args(q, block_tables, context_lens, query_starts, nullptr, out, l.w, tokens, batch, 0, num_heads,
                     num_kv_heads, num_pages, max_pages, scale);
  // Two blocks of rows side by side when the requests have more than one block's rows on average, or when there are few
  // blocks, which make fewer pieces then.  Both forms timed in graphs at 4 / 1 to 64 / 8 heads (us, side by side and
  // not):
  //   33 tokens over 20,000, 4 requests of 32 / 8 heads 98 and 124, 32 of 4 / 1 heads 100 and 126; over 500 20 and 25;
  //   single tokens of as many requests as make 16 blocks, over 500, 3000, 20,000 tokens: 15 and 19, 19 and 22, 52 and
  //   45, of 32 blocks 17 and 20, 25 and 25, 87 and 69, with 1, 2 and 8 KV heads alike: it goes by the blocks, and by
  //   the contexts, which the host does not know;
  //   a prompt of 2048 among 31 single tokens over 2000: 192 and 202 with 32 / 8 heads, 46 and 53 with 4 / 1; where the
  //   average misleads (700 among 63 over 3000, 16 / 1 heads) 50 and 43.
  if (tokens > batch * a.TB || batch * num_kv_heads <= 16) return launch_pt<true, 1>(a, k_cache, v_cache, stream);
  return launch_pt<false, 1>(a, k_cache, v_cache, stream);
}

int launch_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache, const int* block_tables,
                                   const int* context_lens, const int* group_starts, const int* prefix_lens, void* out,
                                   void* workspace, int64_t batch, int64_t groups, int64_t num_heads,
                                   int64_t num_kv_heads, int64_t num_pages, int64_t max_pages, float scale,
                                   cudaStream_t stream) {
  const PtLayout l = pt_shared_layout(static_cast<char*>(workspace), batch, groups, num_heads, num_kv_heads);
  // without groups nothing is read through these two
  const int* prefix = groups > 0 ? prefix_lens : context_lens;
  PtArgs a = pt_args(q, block_tables, context_lens, group_starts, prefix, out, l.w, batch, batch, groups, num_heads,
                     num_kv_heads, num_pages, max_pages, scale);
  return launch_pt<false, 2>(a, k_cache, v_cache, stream);
}

}  // namespace nv4
