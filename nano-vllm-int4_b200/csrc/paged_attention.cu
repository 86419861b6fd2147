// Operators of requests that share cached tokens, over the paged BF16 cache of
// attention.cu ([pages, 256, Hkv, 128]): the append that writes it from q, k and
// v of their own, the attention of prompts over what their requests have cached,
// and the decode attention of a batch whose requests share a prefix's pages.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kPaD = 128;
constexpr int kPaPage = 256;

// ------------------------------------------------------------ append
// Sixteen lanes per row (one head of one token), eight channels (16 bytes) a lane.
// With y = x * rsqrt(mean(x^2) + eps) * w (or x without a norm), channels c and c +
// R/2 of the first R are rotated, (a, b) -> (a cos - b sin, b cos + a sin); FP32
// throughout, one rounding to BF16.  The lane of channel c + R/2 is R/16 lanes on.
// A CTA takes a token, its half warps the heads in turn, so that cos and sin are
// loaded once a lane; four rows are in flight a half warp.  Bound by HBM for long
// prompts, by launch and one chain of loads (position, cos) for few tokens.
struct AppendArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q_weight;
  const uint16_t* k_weight;
  const float* cos_sin;
  const int64_t* positions;
  const int* slots;
  uint16_t* q_out;
  uint16_t* k_cache;
  uint16_t* v_cache;
  int64_t tokens, q_stride, k_stride, v_stride, max_position, num_slots;
  int Hq, Hkv, half_lanes;  // half_lanes: R / 16
  float eps;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendRows = 4;  // rows in flight of a half warp

__device__ __forceinline__ void unpack8(const uint4& r, float (&x)[8]) {
  x[0] = bf16lo_to_f32(r.x), x[1] = bf16hi_to_f32(r.x), x[2] = bf16lo_to_f32(r.y), x[3] = bf16hi_to_f32(r.y);
  x[4] = bf16lo_to_f32(r.z), x[5] = bf16hi_to_f32(r.z), x[6] = bf16lo_to_f32(r.w), x[7] = bf16hi_to_f32(r.w);
}

__global__ void __launch_bounds__(kAppendThreads) append_kv_kernel(const AppendArgs p) {
  const int half = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int heads = p.Hq + 2 * p.Hkv, hl = p.half_lanes;
  const bool first = lane < hl, turned = lane < 2 * hl;
  const int partner = (threadIdx.x & 16) + (first ? lane + hl : lane - hl);
  float qw[8], kw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qw[i] = kw[i] = 1.0f;
  if (p.q_weight) unpack8(__ldg(reinterpret_cast<const uint4*>(p.q_weight) + lane), qw);
  if (p.k_weight) unpack8(__ldg(reinterpret_cast<const uint4*>(p.k_weight) + lane), kw);
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const int64_t pos = p.positions[t];
    const int64_t slot = p.slots ? p.slots[t] : -1;
    const bool known = pos >= 0 && pos < p.max_position;
    if (threadIdx.x == 0) {
      if (!known) record_index_error(kErrBadPosition);
      if (slot >= p.num_slots) record_index_error(kErrBadSlot);
    }
    const bool store = slot >= 0 && slot < p.num_slots;
    float c[8], s[8];
    {
      const int at = (first ? lane : lane - hl) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = 1.0f, s[i] = 0.0f;
      if (turned && known) {
        const float4* row = reinterpret_cast<const float4*>(p.cos_sin + pos * (16 * hl) + at);
        const float4 c0 = __ldg(row), c1 = __ldg(row + 1), s0 = __ldg(row + 2 * hl), s1 = __ldg(row + 2 * hl + 1);
        c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
        s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
        if (first) {
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i] = -s[i];
        }
      }
      if (!known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = __int_as_float(0x7FFFFFFF);
      }
    }
    for (int h0 = half; h0 < heads; h0 += kAppendRows * (kAppendThreads / 16)) {
      uint4 raw[kAppendRows];
#pragma unroll
      for (int j = 0; j < kAppendRows; ++j) {
        const int h = h0 + j * (kAppendThreads / 16);
        if (h >= heads) continue;
        const uint16_t* src = h < p.Hq           ? p.q + t * p.q_stride + h * kPaD
                              : h < p.Hq + p.Hkv ? p.k + t * p.k_stride + (h - p.Hq) * kPaD
                                                 : p.v + t * p.v_stride + (h - p.Hq - p.Hkv) * kPaD;
        raw[j] = *(reinterpret_cast<const uint4*>(src) + lane);
      }
#pragma unroll
      for (int j = 0; j < kAppendRows; ++j) {
        const int h = h0 + j * (kAppendThreads / 16);
        const bool live = h < heads;  // the two rows of a warp may differ: every lane takes part in the shuffles
        const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
        if (!__any_sync(0xffffffffu, live)) break;
        float x[8];
        unpack8(live ? raw[j] : make_uint4(0, 0, 0, 0), x);
        const bool normed = is_q ? p.q_weight != nullptr : p.k_weight != nullptr;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int m = 8; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const float r = normed ? rsqrtf(ss * (1.0f / kPaD) + p.eps) : 1.0f;
        uint32_t packed[4];
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = x[i] * r * (is_q ? qw[i] : kw[i]);
          const float b = __shfl_sync(0xffffffffu, a, partner);
          y[i] = turned ? fmaf(a, c[i], b * s[i]) : a * c[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 o = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
          packed[i] = *reinterpret_cast<const uint32_t*>(&o);
        }
        if (!live) continue;
        const uint4 out = is_v ? raw[j] : make_uint4(packed[0], packed[1], packed[2], packed[3]);
        if (is_q) {
          *(reinterpret_cast<uint4*>(p.q_out + (t * p.Hq + h) * kPaD) + lane) = out;
        } else if (store) {
          const int kh = h - p.Hq - (is_v ? p.Hkv : 0);
          *(reinterpret_cast<uint4*>((is_v ? p.v_cache : p.k_cache) + (slot * p.Hkv + kh) * kPaD) + lane) = out;
        }
      }
    }
  }
}

int launch_append_kv(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                     const float* cos_sin, const int64_t* positions, const int* slot_mapping, void* q_out,
                     void* k_cache, void* v_cache, int64_t tokens, int64_t num_heads, int64_t num_kv_heads,
                     int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t rotary_dim, int64_t num_pages,
                     int64_t max_position, float eps, cudaStream_t stream) {
  AppendArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_weight = static_cast<const uint16_t*>(q_weight);
  a.k_weight = static_cast<const uint16_t*>(k_weight);
  a.cos_sin = cos_sin;
  a.positions = positions;
  a.slots = slot_mapping;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.tokens = tokens;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.max_position = max_position;
  a.num_slots = num_pages * kPaPage;
  a.Hq = q ? static_cast<int>(num_heads) : 0;
  a.Hkv = static_cast<int>(num_kv_heads);
  a.half_lanes = static_cast<int>(rotary_dim / 16);
  a.eps = eps;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(tokens, int64_t(1) << 30));
  return launch_kernel(append_kv_kernel, dim3(grid), dim3(kAppendThreads), 0, stream, false, a);
}

}  // namespace nv4
