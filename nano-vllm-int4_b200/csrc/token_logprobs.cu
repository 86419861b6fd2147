// Log-probabilities of given tokens from their logits, with the tokens' ranks,
// the distribution's entropy and the k most likely alternatives.
//
// For a row x of V logits, with a reference m at most 1 below the maximum, d = x -
// m, S = sum exp(d) and W = sum exp(d) d:
//   logprob(t) = d_t - log S      rank(t) = 1 + #{x > x_t}
//   entropy    = log S - W / S
// (a reference far below the maximum would cost precision: both terms of the
// entropy grow with the distance.  Folding x log2(e) - m log2(e) into one FMA
// saves 3% on 1024 rows but the maximum's own exponential is then not 1.)
// Alternatives are ordered by logit, ties to the lowest index.
//
// One pass over the logits, bound by HBM where there are many rows, with the
// exponential unit (16 a cycle and SM) next.  A warp takes chunks of 512
// contiguous logits, 16 a lane, and moves its reference when a chunk's maximum
// exceeds it by more than 1: that happens a few times a row for the warp, while
// every lane's own maximum would move in most chunks for some lane.  The rank
// costs one comparison with the chunk's maximum unless that exceeds the token's
// logit.  The alternatives cost a
// maximum per chunk and per lane in that pass: the k-th largest maximum of 64
// groups of lanes bounds the k-th largest logit from below (k logits reach it), so
// the few chunks whose maximum reaches it are read again (from L2), the logits
// that do are collected (about k, unless many are equal) and each one's rank is
// counted.
//
// With few rows a row is split over several CTAs, whose results a second kernel
// joins.
//
// Measured: 1024 BF16 rows of 151936 56 us = 5.6 TB/s (0.86 of the measured copy
// rate; 65 us with 5 alternatives, 72 us with 20), 48 FP32 rows of 100003 with 20
// alternatives 15 us, one row with 5 alternatives 11 us (two launches' latency).
#include <cfloat>

#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpChunk = 512;
constexpr int kLpLane = kLpChunk / 32;  // logits of a chunk that a lane takes
constexpr int kLpMaxTop = NV4_LOGPROB_MAX_TOP;
constexpr int kLpMaxChunks = 2048;    // of a CTA: their maxima are held in shared memory
constexpr int kLpCtasPerSm = 4;
constexpr int kLpRingBytes = 4096;    // of a warp: 4 BF16 or 2 FP32 chunks in flight
constexpr int kLpMaxFound = 512;      // logits that reach the alternatives' threshold; more take another way
constexpr int kLpMaxSplits = 64;
static_assert(NV4_LOGPROB_MAX_VOCAB / kLpChunk / kLpMaxChunks < kLpMaxSplits, "the longest row's parts");
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

// Statistics of a set of logits relative to m; m = -inf and S = W = 0 for none
// above -inf.  From |m| = 2^31 on, the next lower FP32 number is 128 or more away
// (256 but for 2^31 itself) and its exponential is 0: S is then the number of logits
// equal to the maximum m, W 0.  Below, m - 110 rounds to a number under m.
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

// The 16 logits of a lane in a chunk: twice 8 consecutive BF16 or four times 4
// FP32 elements.  `base` is the row's start rounded down to 16 bytes, the row's own
// elements are base[lo .. hi); what lies outside is not read and counts as -inf.
__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const uint16_t* p) { return bf16_bits_to_f32(__ldg(p)); }

template <typename T>
struct LaneOf {
  static constexpr int kVec = 16 / sizeof(T), kVecs = kLpLane / kVec;
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
__device__ __forceinline__ void unpack_chunk(const uint4 (&raw)[LaneOf<T>::kVecs], float (&x)[kLpLane]) {
#pragma unroll
  for (int v = 0; v < LaneOf<T>::kVecs; ++v) {
    const uint32_t w[4] = {raw[v].x, raw[v].y, raw[v].z, raw[v].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[4 * v + i] = __uint_as_float(w[i]);
      } else {
        x[8 * v + 2 * i] = bf16lo_to_f32(w[i]);
        x[8 * v + 2 * i + 1] = bf16hi_to_f32(w[i]);
      }
    }
  }
}

__device__ __forceinline__ bool is_big(float m) { return fabsf(m) >= 0x1p31f; }

// Moves statistics from their reference to the larger m.
__device__ __forceinline__ void move_stat(float& s, float& w, float from, float m) {
  if (from == m) return;
  const float d = from - m, f = is_big(from) || is_big(m) ? 0.0f : ex2(d * kLog2e);
  w = f > 0.0f ? f * fmaf(d, s, w) : 0.0f;
  s = f > 0.0f ? f * s : 0.0f;
}
__device__ __forceinline__ LogprobStat join_stats(LogprobStat a, LogprobStat b) {
  const float m = fmaxf(a.m, b.m);
  move_stat(a.s, a.w, a.m, m);
  move_stat(b.s, b.w, b.m, m);
  return {m, a.s + b.s, a.w + b.w, a.above + b.above};
}
// Joins the lanes' statistics (in lane 0); `lanes` of them, a power of two.
__device__ __forceinline__ LogprobStat warp_join(LogprobStat t, int lanes) {
  for (int o = lanes >> 1; o >= 1; o >>= 1) {
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
__device__ __forceinline__ float warp_max(float x) {
  float d;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(x));
  return d;
}

// The k largest of n keys in shared memory, falling, to `out` (left as it is
// where there are fewer): every thread counts the keys above its own.  Keys differ, but for 0.
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int k, uint64_t* out, int tid) {
  for (int i = tid; i < n; i += kLpThreads) {
    const uint64_t mine = keys[i];
    int rank = 0;
    int j = 0;
    for (; j + 8 <= n; j += 8)
#pragma unroll
      for (int u = 0; u < 8; ++u) rank += keys[j + u] > mine;
    for (; j < n; ++j) rank += keys[j] > mine;
    if (mine != 0 && rank < k) out[rank] = mine;
  }
}

// The k largest keys of n <= 64 falling lists of k keys, `stride` apart in shared
// memory, as a warp's list: k times the largest of the lists' heads.
__device__ __forceinline__ uint64_t select_top(const uint64_t* lists, int stride, int n, int k, int lane) {
  const uint64_t *a = lists + lane * stride, *b = a + 32 * stride;
  uint64_t head_a = lane < n ? *a : 0, head_b = lane + 32 < n ? *b : 0, list = 0;
  const uint64_t *end_a = a + k, *end_b = b + k;
  for (int i = 0; i < k; ++i) {
    const uint64_t head = head_a > head_b ? head_a : head_b;
    const uint32_t high = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(head >> 32));
    const uint32_t low =
        __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(head >> 32) == high ? static_cast<uint32_t>(head) : 0);
    const uint64_t key = static_cast<uint64_t>(high) << 32 | low;
    if (key == 0) break;
    if (lane == i) list = key;
    if (head_a == key) head_a = ++a < end_a ? *a : 0;
    else if (head_b == key) head_b = ++b < end_b ? *b : 0;
  }
  return list;
}

// A row's results from its statistics and its list of keys (one warp).
__device__ __forceinline__ void finish_row(const LogprobArgs& p, int64_t row, float xt, bool given,
                                           const LogprobStat& t, bool nan, uint64_t list, int lane) {
  const bool none = nan || t.m == INFINITY, empty = t.m == -INFINITY;
  const float log_s = logf(t.s);
  if (lane == 0) {
    p.logprobs[row] = !given ? 0.0f : none ? NAN : empty ? -INFINITY : (xt - t.m) - log_s;
    p.ranks[row] = given ? t.above + 1 : 0;
    p.entropy[row] = none ? NAN : empty ? 0.0f : log_s - t.w / t.s;
  }
  if (lane < p.top_k) {
    p.top_logprobs[row * p.top_k + lane] = !list ? -INFINITY : none ? NAN : (key_logit(list) - t.m) - log_s;
    p.top_ids[row * p.top_k + lane] = list ? static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(list)) : -1;
  }
}

// The statistics that a warp gathers: the reference is the warp's, the sums and the
// count are the lanes'.
template <typename T>
struct WarpStat {
  float m, limit, floor;  // reference, m + 1; m - 110 or less, whose exponential is 0 (m itself for a big one)
  uint64_t s = 0, w = 0;  // pairs of FP32: even and odd elements
  float above = 0.0f;  // whole numbers below 2^24
  bool nan = false;

  __device__ __forceinline__ WarpStat() { refer(sizeof(T) == 4 ? -FLT_MAX : -0x1.fep127f); }  // the lowest value
  __device__ __forceinline__ void refer(float to) {
    m = to;
    limit = to + 1.0f;
    floor = to - 110.0f;
    if constexpr (sizeof(T) == 2) floor = __bfloat162float(__float2bfloat16_rd(floor));
  }

  // The chunk's logits; returns the lane's maximum (NaN aside).
  __device__ __forceinline__ float add(uint4 (&raw)[LaneOf<T>::kVecs], float xt) {
    constexpr int kWords = 4 * LaneOf<T>::kVecs;
    uint32_t* word = reinterpret_cast<uint32_t*>(&raw[0]);
    float x[kLpLane], top;
    if constexpr (sizeof(T) == 2) {
      uint32_t a = word[0];
#pragma unroll
      for (int i = 1; i < kWords; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(word[i]));
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(bf16lo_to_f32(a)), "f"(bf16hi_to_f32(a)));
    } else {
      unpack_chunk<T>(raw, x);
      top = x[0];
#pragma unroll
      for (int e = 1; e < kLpLane; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(x[e]));
    }
    if (__any_sync(0xffffffffu, !(top <= limit))) {
      if (top != top) {
        nan = true;
        unpack_chunk<T>(raw, x);
        top = -INFINITY;
#pragma unroll
        for (int e = 0; e < kLpLane; ++e) top = fmaxf(top, x[e]);
      }
      const uint32_t order = __reduce_max_sync(0xffffffffu, logit_order(top));
      const float most = key_logit(static_cast<uint64_t>(order) << 32);
      if (order != 0 && most > m) {
        float s0, s1, w0, w1;
        unpair(s, s0, s1);
        unpair(w, w0, w1);
        move_stat(s0, w0, m, most);
        move_stat(s1, w1, m, most);
        s = pair(s0, s1);
        w = pair(w0, w1);
        refer(most);
      }
    }
    if (top > xt) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t t = __float_as_uint(xt), tt = t | (t >> 16);
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          uint32_t g;  // 1.0 or 0.0 in either half
          asm("set.gt.bf16x2.bf16x2 %0, %1, %2;" : "=r"(g) : "r"(word[i]), "r"(tt));
          asm("add.bf16x2 %0, %0, %1;" : "+r"(n) : "r"(g));
        }
        above += bf16lo_to_f32(n) + bf16hi_to_f32(n);
      } else {
        float n = 0.0f;
#pragma unroll
        for (int e = 0; e < kLpLane; ++e) n += x[e] > xt ? 1.0f : 0.0f;
        above += n;
      }
    }
    // Clamped to the floor, d stays finite (0 * -inf would be NaN) and its exponential 0.
    if constexpr (sizeof(T) == 2) {
      const uint32_t f = __float_as_uint(floor), ff = f | (f >> 16);  // floor is a BF16 number
#pragma unroll
      for (int i = 0; i < kWords; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(word[i]) : "r"(ff));
      unpack_chunk<T>(raw, x);
    } else {
#pragma unroll
      for (int e = 0; e < kLpLane; ++e) x[e] = fmaxf(x[e], floor);
    }
    // Two at a time: the packed FP32 operations halve the issue slots.
    const uint64_t minus_m = pair(-m, -m), log2e = pair(kLog2e, kLog2e);
#pragma unroll
    for (int e = 0; e < kLpLane; e += 2) {
      const uint64_t d = add2(pair(x[e], x[e + 1]), minus_m);
      float y0, y1;
      unpair(mul2(d, log2e), y0, y1);
      const uint64_t g = pair(ex2(y0), ex2(y1));
      s = add2(s, g);
      w = fma2(g, d, w);
    }
    return top;
  }
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) token_logprobs_kernel(const LogprobArgs p) {
  // The warps' rings of chunks in flight; after the pass the collected keys and the lists.
  __shared__ __align__(16) uint8_t ring[kLpWarps * kLpRingBytes];
  __shared__ float maxima[kLpMaxChunks];
  uint64_t* found = reinterpret_cast<uint64_t*>(ring);                           // [kLpMaxFound]
  uint64_t(*lists)[32] = reinterpret_cast<uint64_t(*)[32]>(found + kLpMaxFound);  // [kLpWarps]
  uint64_t* sorted = lists[kLpWarps];                                            // [kLpMaxTop]
  static_assert((kLpMaxFound + (kLpWarps + 1) * 32) * 8 <= kLpWarps * kLpRingBytes, "they fit");
  __shared__ float lane_max[kLpWarps][32];
  __shared__ float group_max[64];
  __shared__ LogprobStat stats[kLpWarps];
  __shared__ float bound;
  __shared__ int num_found;
  constexpr int kVecs = LaneOf<T>::kVecs, kVec = LaneOf<T>::kVec;
  constexpr int kDepth = kLpRingBytes / (kLpChunk * sizeof(T));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / p.splits;
  const int split = static_cast<int>(blockIdx.x - row * p.splits);
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int lo = static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (kVec - 1)), hi = lo + p.vocab;
  const T* base = x - lo;
  const int chunks = (hi + kLpChunk - 1) / kLpChunk;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * split / p.splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / p.splits);
  const bool tops = p.top_k > 0;
  if (tid == 0) num_found = 0;

  int64_t target;
  bool given;
  float xt;
  WarpStat<T> st;
  float largest = -INFINITY;  // of the lane's logits
  const auto take = [&](uint4 (&raw)[kVecs], int c) {
    const float top = st.add(raw, xt);
    if (tops) {
      largest = fmaxf(largest, top);
      const float most = warp_max(top);
      if (lane == 0) maxima[c - c0] = most;
    }
  };
  // Only the row's first and last chunk can lie partly outside it.
  const int in0 = c0 * kLpChunk >= lo ? c0 : c0 + 1, in1 = c1 * kLpChunk <= hi ? c1 : c1 - 1;
  // A lane copies into the ring what it reads back itself, so no barrier is needed.
  {
    constexpr int kBytes = kLpChunk * sizeof(T), kDepth = kLpRingBytes / kBytes;
    constexpr int64_t kStep = static_cast<int64_t>(kLpWarps) * kLpChunk;
    const int n = (in1 - in0 - warp + kLpWarps - 1) / kLpWarps;
    const uint32_t slots = smem_u32(ring) + warp * kLpRingBytes + lane * 16;
    const T* at = base + static_cast<int64_t>(in0 + warp) * kLpChunk + lane * kVec;
    const auto issue = [&](uint32_t slot) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) cp_async16(slot + v * 512, at + v * 32 * kVec, 16);
      at += kStep;
    };
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (i < n) issue(slots + i * kBytes);
      cp_async_commit();
    }
    target = p.targets[row];  // these two loads follow one another: behind the copies
    given = target >= 0 && target < p.vocab;
    xt = given ? load_logit(x + target) : INFINITY;
    uint32_t slot = slots, turn = slots + kLpRingBytes;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      cp_async_wait<kDepth - 1>();
      uint4 raw[kVecs];
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(raw[v].x), "=r"(raw[v].y), "=r"(raw[v].z), "=r"(raw[v].w)
                     : "r"(slot + v * 512)
                     : "memory");
      take(raw, in0 + warp + i * kLpWarps);
      if (i + kDepth < n) issue(slot);
      cp_async_commit();
      slot += kBytes;
      if (slot == turn) slot = slots;
    }
    cp_async_wait<0>();
  }
  // The first by warp 0, the last by warp 1 (by warp 0 if it is the first as well).
  int end = -1;
  if (warp == 0 && in0 > c0) end = c0;
  else if (in1 < c1 && warp == (c1 - 1 == c0 ? 0 : 1)) end = c1 - 1;
  if (end >= 0) {
    uint4 raw[kVecs];
    load_chunk<T>(base, end, lane, lo, hi, raw);
    take(raw, end);
  }
  float s, w, s1, w1;
  unpair(st.s, s, s1);
  unpair(st.w, w, w1);
  s += s1;
  w += w1;
  if (is_big(st.m)) {  // the lowest value, if nothing was above it; else the maximum: count what equals it
    s = w = 0.0f;
    for (int c = in0 + warp; c < in1 + kLpWarps; c += kLpWarps) {
      const int own = c < in1 ? c : end;
      if (own < 0) break;
      uint4 raw[kVecs];
      float v[kLpLane];
      load_chunk<T>(base, own, lane, lo, hi, raw);
      unpack_chunk<T>(raw, v);
#pragma unroll
      for (int e = 0; e < kLpLane; ++e) s += v[e] == st.m ? 1.0f : 0.0f;
      if (own == end) break;
    }
    if (!__any_sync(0xffffffffu, s > 0.0f)) st.m = -INFINITY;
  }
  int above = static_cast<int>(st.above);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {  // one reference a warp: plain sums
    s += __shfl_xor_sync(0xffffffffu, s, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
    above += __shfl_xor_sync(0xffffffffu, above, o);
  }
  if (lane == 0) stats[warp] = {st.m, s, w, above};
  if (tops) lane_max[warp][lane] = largest;
  const bool nan = __syncthreads_or(st.nan);

  uint64_t list = 0;
  if (tops) {
    // The top_k-th largest of 64 maxima, each of a lane of four warps.
    if (tid < kLpMaxTop) sorted[tid] = 0;
    if (tid < 64) {
      float g = lane_max[warp * 4][lane];
#pragma unroll
      for (int i = 1; i < 4; ++i) g = fmaxf(g, lane_max[warp * 4 + i][lane]);
      group_max[tid] = g;
      named_barrier_sync(1, 64);
      int rank = 0;
#pragma unroll
      for (int i = 0; i < 64; ++i) rank += group_max[i] > g || (group_max[i] == g && i < tid);
      if (rank == p.top_k - 1) bound = fmaxf(g, -FLT_MAX);  // -inf: no alternative
    }
    __syncthreads();
    // The warp's own chunks that reach it.
    const float least = bound;
    const auto each_picked = [&](const auto& use) {
      for (int i0 = 0; i0 < c1 - c0; i0 += 32 * kLpWarps) {
        const int i = i0 + lane * kLpWarps + warp;
        uint32_t todo = __ballot_sync(0xffffffffu, i < c1 - c0 && maxima[i] >= least);
        for (; todo; todo &= todo - 1) {
          const int c = c0 + i0 + (__ffs(todo) - 1) * kLpWarps + warp;
          uint4 raw[kVecs];
          float v[kLpLane];
          load_chunk<T>(base, c, lane, lo, hi, raw);
          unpack_chunk<T>(raw, v);
#pragma unroll
          for (int e = 0; e < kLpLane; ++e) use(v[e], c * kLpChunk + LaneOf<T>::offset(lane, e) - lo);
        }
      }
    };
    each_picked([&](float v, int index) {
      if (v >= least) {
        const int at = atomicAdd(&num_found, 1);  // in any order: the keys are ordered
        if (at < kLpMaxFound) found[at] = logit_key(logit_order(v), index);
      }
    });
    __syncthreads();
    if (num_found <= kLpMaxFound) {
      rank_keys(found, num_found, p.top_k, sorted, tid);
      __syncthreads();
    } else {  // many equal logits: a sorted list per warp, then the lists' heads
      uint64_t last = 0;  // the warp's top_k-th key
      each_picked([&](float v, int index) {
        const uint64_t k = logit_key(logit_order(v), index);
        uint32_t todo = __ballot_sync(0xffffffffu, v >= least && k > last);
        while (todo) {
          list_insert(list, __shfl_sync(0xffffffffu, k, __ffs(todo) - 1), lane);
          last = __shfl_sync(0xffffffffu, list, p.top_k - 1);
          todo &= todo - 1;
          todo &= __ballot_sync(0xffffffffu, k > last);
        }
      });
      lists[warp][lane] = list;
      __syncthreads();
      if (warp == 0) {
        list = select_top(lists[0], 32, kLpWarps, p.top_k, lane);
        sorted[lane] = list;
        __syncwarp();
      }
    }
    list = lane < p.top_k ? sorted[lane] : 0;
  }
  if (warp != 0) return;
  const LogprobStat t = warp_join(stats[lane & (kLpWarps - 1)], kLpWarps);
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
  __shared__ uint64_t lists[kLpMaxSplits * kLpMaxTop], found[kLpMaxFound], sorted[kLpMaxTop];
  __shared__ int num_found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int64_t target = p.targets[row];
  const bool given = target >= 0 && target < p.vocab;
  const float xt = given ? load_logit(x + target) : INFINITY;
  if (threadIdx.x == 0) num_found = 0;
  if (threadIdx.x < kLpMaxTop) sorted[threadIdx.x] = 0;
  grid_dependency_wait();
  const uint64_t* keys = p.part_keys + row * p.splits * p.top_k;
  for (int i = threadIdx.x; i < p.splits * p.top_k; i += kLpThreads) lists[i] = keys[i];
  LogprobStat t = {-INFINITY, 0.0f, 0.0f, 0};
  bool nan = false;
  if (warp == 0) {
    for (int i = lane; i < p.splits; i += 32) {
      const LogprobPart part = p.parts[row * p.splits + i];
      t = join_stats(t, part.st);
      nan |= part.nan != 0;
    }
    nan = __any_sync(0xffffffffu, nan);
    t = warp_join(t, 32);
  }
  __syncthreads();
  uint64_t list = 0;
  if (p.top_k > 0) {
    // The top_k-th largest of the first few keys of every list (twice as many as
    // wanted) bounds the row's from below; the keys that reach it are ranked.
    const int k = p.top_k, each = min(k, (2 * k + p.splits - 1) / p.splits), n = each * p.splits;
    if (threadIdx.x < n)  // at most 2 k + splits
      found[threadIdx.x] = lists[threadIdx.x / each * k + threadIdx.x % each];
    __syncthreads();
    rank_keys(found, n, k, sorted, threadIdx.x);
    __syncthreads();
    const uint64_t least = max(sorted[k - 1], uint64_t(1));
    for (int i = threadIdx.x; i < p.splits * k; i += kLpThreads)
      if (lists[i] >= least) {
        const int at = atomicAdd(&num_found, 1);
        if (at < kLpMaxFound) found[at] = lists[i];
      }
    __syncthreads();
    if (num_found <= kLpMaxFound) {
      rank_keys(found, num_found, k, sorted, threadIdx.x);
    } else if (warp == 0) {
      sorted[lane] = select_top(lists, k, p.splits, k, lane);
    }
    __syncthreads();
    if (lane < k) list = sorted[lane];
  }
  if (warp == 0) finish_row(p, row, xt, given, t, nan, list, lane);
}

// CTAs of a row: one where the rows alone fill the SMs, else so many that all do,
// with a chunk for every warp at least.  148 are a B200's SMs: the workspace's size
// follows from it, which a caller asks for without a current device.
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
