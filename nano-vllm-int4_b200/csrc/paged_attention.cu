// The append that writes the paged BF16 cache of attention.cu ([pages, 256, Hkv, 128])
// from q, k and v of their own; paged_attention_tc.cu has the two attentions over it.
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
// A half warp takes kRows rows of a token: their loads go out first, then the position
// and slot, then cos and sin, so that two loads in a row are what a warp waits for.
//
// A token's heads are read once and written once: bound by that for long prompts (16,384
// tokens, 32 / 8 heads: 411 MB in 96 us, 4.3 TB/s), by one such chain of loads for a
// decode batch (32 tokens: 2.2 us).  4 CTAs an SM: 3 and 5 take 110 and 115 us there.
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

// Eight BF16 values as four pairs of FP32.
__device__ __forceinline__ void unpack8(const uint4& r, uint64_t (&x)[4]) {
  x[0] = pair(bf16lo_to_f32(r.x), bf16hi_to_f32(r.x)), x[1] = pair(bf16lo_to_f32(r.y), bf16hi_to_f32(r.y));
  x[2] = pair(bf16lo_to_f32(r.z), bf16hi_to_f32(r.z)), x[3] = pair(bf16lo_to_f32(r.w), bf16hi_to_f32(r.w));
}

template <int kRows>
__global__ void __launch_bounds__(kAppendThreads, 4) append_kv_kernel(const AppendArgs p) {
  const int lane = threadIdx.x & 15;
  const int heads = p.Hq + 2 * p.Hkv, hl = p.half_lanes;
  const uint32_t groups = (heads + kRows - 1) / kRows;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x) >> 4;
  // a half warp behind the last row works on it once more (every lane takes part in the shuffles) and stores nothing
  const bool live = unit < p.tokens * groups;
  const int64_t t = live ? unit / groups : p.tokens - 1;
  const int h0 = static_cast<int>(live ? unit - t * groups : 0) * kRows;
  uint4 raw[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int h = min(h0 + j, heads - 1);
    const uint16_t* src = h < p.Hq           ? p.q + t * p.q_stride + h * kPaD
                          : h < p.Hq + p.Hkv ? p.k + t * p.k_stride + (h - p.Hq) * kPaD
                                             : p.v + t * p.v_stride + (h - p.Hq - p.Hkv) * kPaD;
    raw[j] = *(reinterpret_cast<const uint4*>(src) + lane);
  }
  const int64_t pos = p.positions[t];
  const int64_t slot = p.slots[t];
  const bool known = pos >= 0 && pos < p.max_position, store = slot >= 0 && slot < p.num_slots;
  if (live && h0 == 0 && lane == 0) {
    if (!known) record_index_error(kErrBadPosition);
    if (slot >= p.num_slots) record_index_error(kErrBadSlot);
  }
  const bool first = lane < hl, turned = lane < 2 * hl;
  const int partner = (threadIdx.x & 16) + (first ? lane + hl : lane - hl);
  uint64_t c[4], s[4];  // (a, b) -> (a c + b s): one and zero where nothing is turned, NaN at an unknown position
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float one = known ? 1.0f : __int_as_float(0x7FFFFFFF);
    c[i] = pair(one, one), s[i] = 0;
  }
  if (turned && known && h0 < p.Hq + p.Hkv) {
    const ulonglong2* row =
        reinterpret_cast<const ulonglong2*>(p.cos_sin + pos * (16 * hl) + (first ? lane : lane - hl) * 8);
    const ulonglong2 c0 = __ldg(row), c1 = __ldg(row + 1), s0 = __ldg(row + 2 * hl), s1 = __ldg(row + 2 * hl + 1);
    c[0] = c0.x, c[1] = c0.y, c[2] = c1.x, c[3] = c1.y;
    const uint64_t sign = first ? 0x8000000080000000ull : 0;
    s[0] = s0.x ^ sign, s[1] = s0.y ^ sign, s[2] = s1.x ^ sign, s[3] = s1.y ^ sign;
  }
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int h = h0 + j;
    const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
    uint4 out = raw[j];
    if (__any_sync(0xffffffffu, !is_v)) {
      uint64_t x[4];
      unpack8(raw[j], x);
      const uint16_t* weight = is_q ? p.q_weight : p.k_weight;
      if (p.q_weight || p.k_weight) {
        float ss, odd;
        unpair(fma2(x[3], x[3], fma2(x[2], x[2], fma2(x[1], x[1], mul2(x[0], x[0])))), ss, odd);
        ss += odd;
#pragma unroll
        for (int m = 8; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        if (weight) {
          const float r = rsqrtf(ss * (1.0f / kPaD) + p.eps);
          uint64_t w[4];
          unpack8(__ldg(reinterpret_cast<const uint4*>(weight) + lane), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], pair(r, r)), w[i]);
        }
      }
      uint32_t packed[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b, u, v;
        unpair(x[i], a, b);
        const float pa = __shfl_sync(0xffffffffu, a, partner), pb = __shfl_sync(0xffffffffu, b, partner);
        unpair(turned ? fma2(x[i], c[i], mul2(pair(pa, pb), s[i])) : mul2(x[i], c[i]), u, v);
        const __nv_bfloat162 y = __floats2bfloat162_rn(u, v);
        packed[i] = *reinterpret_cast<const uint32_t*>(&y);
      }
      if (!is_v) out = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    }
    if (!live || h >= heads) continue;
    if (is_q) {
      *(reinterpret_cast<uint4*>(p.q_out + (t * p.Hq + h) * kPaD) + lane) = out;
    } else if (store) {
      const int kh = h - p.Hq - (is_v ? p.Hkv : 0);
      *(reinterpret_cast<uint4*>((is_v ? p.v_cache : p.k_cache) + (slot * p.Hkv + kh) * kPaD) + lane) = out;
    }
  }
}

template <int kRows>
static int launch_append_rows(const AppendArgs& a, cudaStream_t stream) {
  const int64_t units = a.tokens * ((a.Hq + 2 * a.Hkv + kRows - 1) / kRows);
  const int64_t blocks = (units * 16 + kAppendThreads - 1) / kAppendThreads;
  return launch_kernel(append_kv_kernel<kRows>, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0, stream,
                       false, a);
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
  // One row a half warp while there are few (a shorter chain; 32 / 8 heads, 128 tokens: 2.6 us, 3.5 with four), else
  // four (fewer loads of cos and sin; 301 tokens: 4.2 us, 4.5 with one, 3.9 with two; 2400: 16.1, 24.7, 18.4 us).
  const int64_t rows = tokens * (a.Hq + 2 * num_kv_heads);
  return rows <= 8192 ? launch_append_rows<1>(a, stream) : launch_append_rows<4>(a, stream);
}

}  // namespace nv4
