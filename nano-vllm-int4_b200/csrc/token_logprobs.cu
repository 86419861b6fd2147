// Log-probabilities of given tokens from their logits, with the tokens' ranks,
// the distribution's entropy and the k most likely alternatives.
//
// For a row x of V logits with maximum m, S = sum exp(x - m) and W = sum
// exp(x - m) (x - m):
//   logprob(t) = x_t - m - log S          rank(t) = 1 + #{x > x_t}
//   entropy    = log S - W / S            (both terms >= 0: nothing cancels)
// Alternatives are ordered by logit, ties to the lowest index.
//
// One pass over the logits, bound by HBM where there are many rows.  A warp
// takes chunks of 256 contiguous logits, eight a lane; every lane keeps its own
// running (m, S, W).  The rank costs one comparison with the chunk's maximum
// unless that exceeds the token's logit.  The alternatives cost one maximum per
// chunk in that pass: the k largest elements lie in the k chunks with the largest
// maxima (for any other chunk there are k elements above all of it), so after the
// pass a threshold is found among the maxima, the few chunks that reach it are
// read again (from L2) and their elements above it sorted.
//
// With few rows a row is split over several CTAs, whose results a second kernel
// joins.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpChunk = 256;
constexpr int kLpMaxTop = NV4_LOGPROB_MAX_TOP;
constexpr int kLpMaxChunks = 2048;    // of a CTA: their maxima are held in shared memory
constexpr int kLpCtasPerSm = 4;
constexpr int kLpMaxSplits = 64;      // but for rows whose chunks need more
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobArgs {
  const void* logits;
  const int64_t* targets;
  float* logprobs;
  int64_t* ranks;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  struct LogprobPart* parts;  // [rows][splits]
  uint64_t* part_keys;        // [rows][splits][top_k]
  int64_t row_stride;
  int rows, vocab, top_k, splits;
};

// Statistics of a set of logits: m = -inf and S = W = 0 for none above -inf.
struct LogprobStat {
  float m, s, w;
  int above;
};
struct LogprobPart {
  LogprobStat st;
  int nan;
};

// Order of the alternatives as one integer: the logit's order, then the lowest
// index.  0 is below every candidate (-inf and NaN are none).
__device__ __forceinline__ uint32_t logit_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 orders as 0
  const uint32_t order = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x > -INFINITY ? order : 0;
}
__device__ __forceinline__ uint64_t logit_key(uint32_t order, int index) {
  return order ? (static_cast<uint64_t>(order) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(index)) : 0;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t order = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? (order & 0x7FFFFFFFu) : ~order);
}

// The eight logits of a lane in a chunk: 8 consecutive BF16 or twice 4 FP32
// elements.  `base` is the row's start rounded down to 16 bytes, the row's own
// elements are base[lo .. hi); what lies outside is not read and counts as -inf.
__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const uint16_t* p) { return bf16_bits_to_f32(__ldg(p)); }

template <typename T>
struct LaneOf {
  static constexpr int kVec = 16 / sizeof(T), kVecs = 8 / kVec;
  static __device__ __forceinline__ int offset(int lane, int e) {  // of element e of a lane within the chunk
    return (e / kVec) * 32 * kVec + lane * kVec + e % kVec;
  }
};

template <typename T>
__device__ __forceinline__ void load_chunk(const T* base, int chunk, int lane, int lo, int hi, uint4 (&raw)[LaneOf<T>::kVecs]) {
  using L = LaneOf<T>;
#pragma unroll
  for (int v = 0; v < L::kVecs; ++v) {
    const int at = chunk * kLpChunk + L::offset(lane, v * L::kVec);
    if (at >= lo && at + L::kVec <= hi) {
      raw[v] = __ldg(reinterpret_cast<const uint4*>(base + at));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          w[i] = at + i >= lo && at + i < hi ? __ldg(reinterpret_cast<const uint32_t*>(base + at + i)) : 0xFF800000u;
        } else {
          const int a = at + 2 * i;
          const uint32_t l = a >= lo && a < hi ? __ldg(reinterpret_cast<const uint16_t*>(base) + a) : 0xFF80u;
          const uint32_t h =
              a + 1 >= lo && a + 1 < hi ? __ldg(reinterpret_cast<const uint16_t*>(base) + a + 1) : 0xFF80u;
          w[i] = l | (h << 16);
        }
      }
      raw[v] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void unpack_chunk(const uint4 (&raw)[LaneOf<T>::kVecs], float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      x[4 * v] = __uint_as_float(raw[v].x), x[4 * v + 1] = __uint_as_float(raw[v].y);
      x[4 * v + 2] = __uint_as_float(raw[v].z), x[4 * v + 3] = __uint_as_float(raw[v].w);
    }
  } else {
    const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = bf16lo_to_f32(w[i]), x[2 * i + 1] = bf16hi_to_f32(w[i]);
  }
}

// The statistics of a joined with those of b.
__device__ __forceinline__ LogprobStat join_stats(const LogprobStat& a, const LogprobStat& b) {
  LogprobStat r;
  r.m = fmaxf(a.m, b.m);
  r.above = a.above + b.above;
  r.s = r.w = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const LogprobStat& t = i ? b : a;
    if (t.m == r.m) {
      r.s += t.s, r.w += t.w;
    } else if (t.m > -INFINITY) {
      const float d = t.m - r.m, f = exp2f(d * kLog2e);
      if (f > 0.0f) r.s = fmaf(f, t.s, r.s), r.w = fmaf(f, fmaf(d, t.s, t.w), r.w);
    }
  }
  return r;
}
__device__ __forceinline__ LogprobStat warp_join(LogprobStat t) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    LogprobStat u;
    u.m = __shfl_xor_sync(0xffffffffu, t.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, t.s, o);
    u.w = __shfl_xor_sync(0xffffffffu, t.w, o);
    u.above = __shfl_xor_sync(0xffffffffu, t.above, o);
    t = join_stats(t, u);
  }
  return t;
}

// A warp's list of the largest keys, falling over the lanes.
__device__ __forceinline__ void list_insert(uint64_t& list, uint64_t key, int lane) {
  const int pos = __popc(__ballot_sync(0xffffffffu, list > key));
  const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
  list = lane < pos ? list : lane == pos ? key : up;
}
// The 32 largest of two such lists.
__device__ __forceinline__ uint64_t list_merge(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  a = a > r ? a : r;  // bitonic
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const uint64_t t = __shfl_xor_sync(0xffffffffu, a, o);
    a = ((lane & o) == 0) == (a > t) ? a : t;
  }
  return a;
}

// A row's results from its statistics and its list of keys (one warp).
__device__ __forceinline__ void finish_row(const LogprobArgs& p, int64_t row, float xt, bool given,
                                           const LogprobStat& t, bool nan, uint64_t list, int lane) {
  const bool empty = t.m == -INFINITY && !nan;
  const float m = nan ? NAN : t.m, log_s = logf(t.s);
  if (lane == 0) {
    p.logprobs[row] = !given ? 0.0f : empty ? -INFINITY : (xt - m) - log_s;
    p.ranks[row] = given ? t.above + 1 : 0;
    p.entropy[row] = empty ? 0.0f : nan ? NAN : log_s - t.w / t.s;
  }
  if (lane < p.top_k) {
    p.top_logprobs[row * p.top_k + lane] = list ? (key_logit(list) - m) - log_s : -INFINITY;
    p.top_ids[row * p.top_k + lane] = list ? static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(list)) : -1;
  }
}

// A logit below which exp(x - m) is 0 in FP32 whatever it is, so that clamping to
// it keeps x - m finite (0 * -inf would be NaN); below m where m - 110 is m.
// -inf where there is none (m is the type's lowest value).
template <typename T>
__device__ __forceinline__ float logit_floor(float m) {
  float l = m - 110.0f;
  if constexpr (sizeof(T) == 4) {
    return l < m ? l : nextafterf(m, -INFINITY);
  } else {
    l = __bfloat162float(__float2bfloat16_rd(l));
    if (l < m) return l;
    const uint32_t bits = __float_as_uint(m) >> 16;  // |m| is large: the BF16 number below it
    return __uint_as_float((m > 0.0f ? bits - 1 : bits + 1) << 16);
  }
}

template <typename T>
struct LaneStat {
  LogprobStat t;
  float floor;  // of t.m
  bool nan;

  // The chunk's eight logits; returns their maximum (NaN aside).
  __device__ __forceinline__ float add(uint4 (&raw)[LaneOf<T>::kVecs], float xt) {
    float x[8], top;
    if constexpr (sizeof(T) == 2) {
      uint32_t a, b;
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(raw[0].x), "r"(raw[0].y));
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(raw[0].z), "r"(raw[0].w));
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(bf16lo_to_f32(a)), "f"(bf16hi_to_f32(a)));
    } else {
      unpack_chunk<T>(raw, x);
      top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(x[e]));
    }
    if (top != top) {
      nan = true;
      unpack_chunk<T>(raw, x);
      top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
    }
    if (top > xt) {
      unpack_chunk<T>(raw, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) t.above += x[e] > xt;
    }
    if (top > t.m) {
      if (t.m > -INFINITY) {
        const float d = t.m - top, f = exp2f(d * kLog2e);
        if (f > 0.0f) t.w = f * fmaf(d, t.s, t.w), t.s *= f;
        else t.w = t.s = 0.0f;
      }
      t.m = top;
      floor = logit_floor<T>(top);
    }
    if (t.m == -INFINITY) return top;
    if (floor > -INFINITY) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t f = __float_as_uint(floor), ff = f | (f >> 16);  // floor is a BF16 number
        uint32_t* w = reinterpret_cast<uint32_t*>(&raw[0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(ff));
        unpack_chunk<T>(raw, x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaxf(x[e], floor);
      }
      float s0 = 0.0f, s1 = 0.0f, w0 = 0.0f, w1 = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float d0 = x[e] - t.m, d1 = x[e + 1] - t.m;
        const float e0 = ex2(d0 * kLog2e), e1 = ex2(d1 * kLog2e);
        s0 += e0, s1 += e1;
        w0 = fmaf(e0, d0, w0), w1 = fmaf(e1, d1, w1);
      }
      t.s += s0 + s1;
      t.w += w0 + w1;
    } else {  // the maximum is the type's lowest value: the others are it or -inf
      unpack_chunk<T>(raw, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) t.s += x[e] == t.m ? 1.0f : 0.0f;
    }
    return top;
  }
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) token_logprobs_kernel(const LogprobArgs p) {
  __shared__ uint32_t maxima[kLpMaxChunks];
  __shared__ int picked[kLpMaxChunks];
  __shared__ uint64_t lists[kLpWarps][32];
  __shared__ uint32_t sorted[kLpWarps][32];
  __shared__ LogprobStat stats[kLpWarps];
  __shared__ uint32_t bound;
  __shared__ int num_picked;
  constexpr int kVecs = LaneOf<T>::kVecs, kVec = LaneOf<T>::kVec;
  constexpr int kAhead = 4 / kVecs;  // chunks a warp loads ahead: 64 bytes a lane
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / p.splits;
  const int split = static_cast<int>(blockIdx.x - row * p.splits);
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int lo = static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (kVec - 1)), hi = lo + p.vocab;
  const T* base = x - lo;
  const int chunks = (hi + kLpChunk - 1) / kLpChunk;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * split / p.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / p.splits);
  const int64_t target = p.targets[row];
  const bool given = target >= 0 && target < p.vocab;
  const float xt = given ? load_logit(x + target) : INFINITY;
  const bool tops = p.top_k > 0;
  if (tid == 0) bound = 0, num_picked = 0;

  LaneStat<T> st;
  st.t.m = -INFINITY, st.t.s = st.t.w = 0.0f, st.t.above = 0;
  st.floor = -INFINITY;
  st.nan = false;
  for (int c = c0 + warp; c < c1; c += kLpWarps * kAhead) {
    uint4 raw[kAhead][kVecs];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (c + u * kLpWarps < c1) load_chunk<T>(base, c + u * kLpWarps, lane, lo, hi, raw[u]);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (c + u * kLpWarps >= c1) break;
      const float top = st.add(raw[u], xt);
      if (tops) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, logit_order(top));
        if (lane == 0) maxima[c + u * kLpWarps - c0] = most;
      }
    }
  }
  st.t = warp_join(st.t);
  if (lane == 0) stats[warp] = st.t;
  const bool nan = __syncthreads_or(st.nan);

  uint64_t list = 0;
  if (tops) {
    // The top_k-th largest of the threads' largest maxima bounds that of the row from
    // below.  Each warp sorts its 32; a key's rank is its lane plus what the others hold above it.
    uint32_t key = 0;
    for (int i = tid; i < c1 - c0; i += kLpThreads) key = max(key, maxima[i]);
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int o = k >> 1; o >= 1; o >>= 1) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, key, o);
        const bool larger = ((lane & o) == 0) == ((lane & k) == 0);  // falling over the lanes
        key = larger ? max(key, other) : min(key, other);
      }
    sorted[warp][lane] = key;
    __syncthreads();
    int rank = lane;
#pragma unroll
    for (int w = 0; w < kLpWarps; ++w) {
      if (w == warp) continue;
      int n = 0;  // keys of warp w before this one: above it, or equal and of an earlier warp
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const uint32_t other = sorted[w][n + o - 1];
        if (other > key || (other == key && w < warp)) n += o;
      }
      if (n == 31) n += sorted[w][31] > key || (sorted[w][31] == key && w < warp);
      rank += n;
    }
    if (rank == p.top_k - 1) bound = key;
    __syncthreads();
    const uint32_t least = max(bound, 1u);  // 0: chunks of nothing but -inf
    for (int i = tid; i < c1 - c0; i += kLpThreads)
      if (maxima[i] >= least) picked[atomicAdd(&num_picked, 1)] = i;  // in any order: the keys are ordered
    __syncthreads();
    const int n = num_picked;
    uint64_t last = 0;  // the warp's top_k-th key
    for (int i = warp; i < n; i += kLpWarps) {
      const int c = c0 + picked[i];
      uint4 raw[kVecs];
      load_chunk<T>(base, c, lane, lo, hi, raw);
      float v[8];
      unpack_chunk<T>(raw, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t order = logit_order(v[e]);
        const uint64_t k = logit_key(order, c * kLpChunk + LaneOf<T>::offset(lane, e) - lo);
        uint32_t todo = __ballot_sync(0xffffffffu, order >= least && k > last);
        while (todo) {
          const int from = __ffs(todo) - 1;
          list_insert(list, __shfl_sync(0xffffffffu, k, from), lane);
          last = __shfl_sync(0xffffffffu, list, p.top_k - 1);
          todo &= todo - 1;
          todo &= __ballot_sync(0xffffffffu, k > last);
        }
      }
    }
    lists[warp][lane] = list;
    __syncthreads();
  }
  if (warp != 0) return;
  if (tops)
    for (int w = 1; w < kLpWarps; ++w) list = list_merge(list, lists[w][lane], lane);
  LogprobStat t;
  t.m = -INFINITY, t.s = t.w = 0.0f, t.above = 0;
  if (lane < kLpWarps) t = stats[lane];
  t = warp_join(t);
  if (p.splits == 1) {
    finish_row(p, row, xt, given, t, nan, list, lane);
  } else {
    if (lane == 0) p.parts[blockIdx.x] = {t, nan};
    if (lane < p.top_k) p.part_keys[static_cast<int64_t>(blockIdx.x) * p.top_k + lane] = list;
  }
}

// Joins the parts of a row; one CTA per row.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_join_kernel(const LogprobArgs p) {
  __shared__ uint64_t lists[kLpWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int64_t target = p.targets[row];
  const bool given = target >= 0 && target < p.vocab;
  const float xt = given ? load_logit(x + target) : INFINITY;
  grid_dependency_wait();
  uint64_t list = 0;
  if (p.top_k > 0) {
    for (int i = warp; i < p.splits; i += kLpWarps) {
      const uint64_t k = lane < p.top_k ? p.part_keys[(row * p.splits + i) * p.top_k + lane] : 0;
      list = i == warp ? k : list_merge(list, k, lane);
    }
    lists[warp][lane] = list;
    __syncthreads();
  }
  if (warp != 0) return;
  if (p.top_k > 0)
    for (int w = 1; w < kLpWarps; ++w) list = list_merge(list, lists[w][lane], lane);
  LogprobStat t;
  t.m = -INFINITY, t.s = t.w = 0.0f, t.above = 0;
  bool nan = false;
  for (int i = lane; i < p.splits; i += 32) {
    const LogprobPart& part = p.parts[row * p.splits + i];
    t = join_stats(t, part.st);
    nan |= part.nan != 0;
  }
  nan = __any_sync(0xffffffffu, nan);
  t = warp_join(t);
  finish_row(p, row, xt, given, t, nan, list, lane);
}

// CTAs of a row: one where the rows alone fill the SMs, else so many that all do,
// with a chunk for every warp at least.
static int64_t logprob_splits(int64_t rows, int64_t vocab) {
  const int64_t chunks = (vocab + kLpChunk - 1) / kLpChunk;
  const int64_t wanted = std::min<int64_t>(kLpCtasPerSm * 148 / rows, std::min<int64_t>(chunks / kLpWarps, kLpMaxSplits));
  return std::max<int64_t>(std::max<int64_t>(wanted, 1), (chunks + kLpMaxChunks) / kLpMaxChunks);
}
int64_t token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top_k) {
  const int64_t splits = logprob_splits(rows, vocab);
  return splits == 1 ? 0 : rows * splits * (static_cast<int64_t>(sizeof(LogprobPart)) + 4 + 8 * top_k);
}

template <typename T>
static int launch_logprobs(const LogprobArgs& a, cudaStream_t stream) {
  const int rc = launch_kernel(token_logprobs_kernel<T>, dim3(static_cast<unsigned>(static_cast<int64_t>(a.rows) * a.splits)),
                               dim3(kLpThreads), 0, stream, false, a);
  if (rc != NV4_OK || a.splits == 1) return rc;
  return launch_kernel(token_logprobs_join_kernel<T>, dim3(a.rows), dim3(kLpThreads), 0, stream, true, a);
}

int launch_token_logprobs(const void* logits, int fp32, const int64_t* targets, float* logprobs, int64_t* ranks,
                          float* entropy, float* top_logprobs, int64_t* top_ids, void* workspace, int64_t rows,
                          int64_t vocab, int64_t row_stride, int64_t top_k, cudaStream_t stream) {
  LogprobArgs a;
  a.logits = logits;
  a.targets = targets;
  a.logprobs = logprobs;
  a.ranks = ranks;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  a.row_stride = row_stride;
  a.rows = static_cast<int>(rows);
  a.vocab = static_cast<int>(vocab);
  a.top_k = static_cast<int>(top_k);
  a.splits = static_cast<int>(logprob_splits(rows, vocab));
  a.part_keys = static_cast<uint64_t*>(workspace);  // first: 8-byte aligned
  a.parts = reinterpret_cast<LogprobPart*>(a.part_keys + rows * a.splits * top_k);
  return fp32 ? launch_logprobs<float>(a, stream) : launch_logprobs<uint16_t>(a, stream);
}

}  // namespace nv4
