// Log-probabilities of given tokens from their logits, with the tokens' ranks,
// the distribution's entropy and the k most likely alternatives.
//
// For a row x of V logits with maximum m and S = sum exp(x - m):
//   logprob(t) = x_t - m - log S          rank(t) = 1 + #{x > x_t}
//   entropy    = log S - sum exp(x - m) (x - m) / S
// (both terms of the entropy are >= 0, so nothing cancels).  Alternatives are
// ordered by logit, ties to the lowest index.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kLpThreads = 256;
constexpr int kLpMaxTop = 32;

struct LogprobArgs {
  const void* logits;
  const int64_t* targets;
  float* logprobs;
  int64_t* ranks;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  int64_t row_stride;
  int rows, vocab, top_k;
};

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const uint16_t* p) { return bf16_bits_to_f32(*p); }

// Order of the alternatives as one integer: the logit's order, then the lowest
// index.  0 is below every candidate (-inf and NaN are none).
__device__ __forceinline__ uint64_t logit_key(float x, int index) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 orders as 0
  const uint32_t order = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x > -INFINITY ? (static_cast<uint64_t>(order) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(index)) : 0;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t order = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? (order & 0x7FFFFFFFu) : ~order);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobArgs p) {
  __shared__ float fbuf[kLpThreads / 32];
  __shared__ float fbuf2[kLpThreads / 32];
  __shared__ int ibuf[kLpThreads / 32];
  __shared__ uint64_t kbuf[kLpThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int64_t target = p.targets[row];
  const bool given = target >= 0 && target < p.vocab;
  const float xt = given ? load_logit(x + target) : INFINITY;

  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < p.vocab; i += kLpThreads) {
    const float v = load_logit(x + i);
    nan |= v != v;
    m = fmaxf(m, v);
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) fbuf[warp] = m;
  nan = __syncthreads_or(nan);
  for (int w = 0; w < kLpThreads / 32; ++w) m = fmaxf(m, fbuf[w]);
  __syncthreads();
  if (nan) m = NAN;
  const bool empty = m == -INFINITY;

  float s = 0.0f, w1 = 0.0f;
  int above = 0;
  for (int i = tid; i < p.vocab; i += kLpThreads) {
    const float v = load_logit(x + i);
    const float d = v - m, e = expf(d);
    s += e;
    if (e > 0.0f) w1 += e * d;
    above += v > xt;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    w1 += __shfl_xor_sync(0xffffffffu, w1, o);
    above += __shfl_xor_sync(0xffffffffu, above, o);
  }
  if (lane == 0) fbuf[warp] = s, fbuf2[warp] = w1, ibuf[warp] = above;
  __syncthreads();
  s = 0.0f, w1 = 0.0f, above = 0;
  for (int w = 0; w < kLpThreads / 32; ++w) s += fbuf[w], w1 += fbuf2[w], above += ibuf[w];
  const float log_s = logf(s);
  if (tid == 0) {
    p.entropy[row] = empty ? 0.0f : log_s - w1 / s;
    p.logprobs[row] = !given ? 0.0f : empty ? -INFINITY : xt - m - log_s;
    p.ranks[row] = given ? above + 1 : 0;
  }
  uint64_t bound = ~0ull;
  for (int k = 0; k < p.top_k; ++k) {
    uint64_t best = 0;
    for (int i = tid; i < p.vocab; i += kLpThreads) {
      const uint64_t key = logit_key(load_logit(x + i), i);
      if (key < bound && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) kbuf[warp] = best;
    __syncthreads();
    for (int w = 0; w < kLpThreads / 32; ++w) best = kbuf[w] > best ? kbuf[w] : best;
    bound = best;
    if (tid == 0) {
      p.top_ids[row * p.top_k + k] = best ? static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(best)) : -1;
      p.top_logprobs[row * p.top_k + k] = best ? key_logit(best) - m - log_s : -INFINITY;
    }
    if (best == 0) bound = 0;
  }
}

int launch_token_logprobs(const void* logits, int fp32, const int64_t* targets, float* logprobs, int64_t* ranks,
                          float* entropy, float* top_logprobs, int64_t* top_ids, int64_t rows, int64_t vocab,
                          int64_t row_stride, int64_t top_k, cudaStream_t stream) {
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
  return launch_kernel(fp32 ? token_logprobs_kernel<float> : token_logprobs_kernel<uint16_t>,
                       dim3(static_cast<unsigned>(rows)), dim3(kLpThreads), 0, stream, false, a);
}

}  // namespace nv4
