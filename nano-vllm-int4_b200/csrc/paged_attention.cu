// The append that writes the paged BF16 cache of attention.cu ([pages, 256, Hkv, 128])
// from q, k and v of their own; paged_attention_tc.cu has the two attentions over it.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kPaD = 128;
constexpr int kPaPage = 256;

// ------------------------------------------------------------ append
// Sixteen lanes per row (one head of one token), eight channels a lane: of the first R four
// and those R/2 on, which are rotated with them, so that no lane needs another's; of the
// rest eight in a row.
// With y = x * rsqrt(mean(x^2) + eps) * w (or x without a norm), channels c and c +
// R/2 of the first R are rotated, (a, b) -> (a cos - b sin, b cos + a sin); FP32
// throughout, one rounding to BF16.
// A half warp takes kRows rows of a token: their loads go out first, then the position
// and slot, then cos and sin, so that two loads in a row are what a warp waits for.
//
// A token's heads are read once and written once: bound by that and by the instructions for
// long prompts (16,384 tokens, 32 / 8 heads: 411 MB in 84 us, 4.9 TB/s, 0.75 instructions a
// cycle and scheduler), by one such chain of loads for a decode batch (32 tokens: 2.1 us).
// 5 CTAs an SM: 4 take 92 us there, 6 104 us.
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

// Two times four BF16 values as pairs of FP32.
__device__ __forceinline__ void unpack8(const uint2& a, const uint2& b, uint64_t (&x)[4]) {
  x[0] = pair(bf16lo_to_f32(a.x), bf16hi_to_f32(a.x)), x[1] = pair(bf16lo_to_f32(a.y), bf16hi_to_f32(a.y));
  x[2] = pair(bf16lo_to_f32(b.x), bf16hi_to_f32(b.x)), x[3] = pair(bf16lo_to_f32(b.y), bf16hi_to_f32(b.y));
}
__device__ __forceinline__ uint32_t pack2(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&y);
}

template <int kRows>
__global__ void __launch_bounds__(kAppendThreads, 5) append_kv_kernel(const AppendArgs p) {
  const int lane = threadIdx.x & 15;
  const int heads = p.Hq + 2 * p.Hkv, hl = p.half_lanes;
  const uint32_t groups = (heads + kRows - 1) / kRows;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x) >> 4;
  // a half warp behind the last row works on it once more (every lane takes part in the shuffles) and stores nothing
  const bool live = unit < p.tokens * groups;
  const int64_t t = live ? unit / groups : p.tokens - 1;
  const int h0 = static_cast<int>(live ? unit - t * groups : 0) * kRows;
  const bool turned = lane < 2 * hl;
  const int at = (turned ? 4 : 8) * lane, at2 = at + (turned ? 8 * hl : 4);  // channels
  uint2 raw[kRows], raw2[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int h = min(h0 + j, heads - 1);
    const uint16_t* src = h < p.Hq           ? p.q + t * p.q_stride + h * kPaD
                          : h < p.Hq + p.Hkv ? p.k + t * p.k_stride + (h - p.Hq) * kPaD
                                             : p.v + t * p.v_stride + (h - p.Hq - p.Hkv) * kPaD;
    raw[j] = *reinterpret_cast<const uint2*>(src + at);
    raw2[j] = *reinterpret_cast<const uint2*>(src + at2);
  }
  const int64_t pos = p.positions[t];
  const int64_t slot = p.slots[t];
  const bool known = pos >= 0 && pos < p.max_position, store = slot >= 0 && slot < p.num_slots;
  if (live && h0 == 0 && lane == 0) {
    if (!known) record_index_error(kErrBadPosition);
    if (slot >= p.num_slots) record_index_error(kErrBadSlot);
  }
  // (a, b) -> (a c - b s, b c + a s); an unknown position makes all of it NaN
  uint64_t c[2], s[2] = {0, 0};
  const float one = known ? 1.0f : __int_as_float(0x7FFFFFFF);
  c[0] = c[1] = pair(one, one);
  if (turned && known && h0 < p.Hq + p.Hkv) {
    const float* row = p.cos_sin + pos * (16 * hl) + at;
    const ulonglong2 cs = __ldg(reinterpret_cast<const ulonglong2*>(row));
    const ulonglong2 sn = __ldg(reinterpret_cast<const ulonglong2*>(row + 8 * hl));
    c[0] = cs.x, c[1] = cs.y, s[0] = sn.x, s[1] = sn.y;
  }
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int h = h0 + j;
    const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
    uint2 out = raw[j], out2 = raw2[j];
    if (__any_sync(0xffffffffu, !is_v)) {
      uint64_t x[4];
      unpack8(raw[j], raw2[j], x);
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
          unpack8(__ldg(reinterpret_cast<const uint2*>(weight + at)),
                  __ldg(reinterpret_cast<const uint2*>(weight + at2)), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], pair(r, r)), w[i]);
        }
      }
      if (turned) {
        constexpr uint64_t kSigns = 0x8000000080000000ull;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint64_t a = x[i], b = x[i + 2];
          x[i] = fma2(a, c[i], mul2(b, s[i] ^ kSigns));
          x[i + 2] = fma2(b, c[i], mul2(a, s[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], c[0]);
      }
      if (!is_v) out = make_uint2(pack2(x[0]), pack2(x[1])), out2 = make_uint2(pack2(x[2]), pack2(x[3]));
    }
    if (!live || h >= heads) continue;
    uint16_t* dst = nullptr;
    if (is_q) dst = p.q_out + (t * p.Hq + h) * kPaD;
    else if (store) dst = (is_v ? p.v_cache : p.k_cache) + (slot * p.Hkv + (h - p.Hq - (is_v ? p.Hkv : 0))) * kPaD;
    if (!dst) continue;
    *reinterpret_cast<uint2*>(dst + at) = out;
    *reinterpret_cast<uint2*>(dst + at2) = out2;
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
  // One row a half warp while there are few (a shorter chain), else four (fewer loads of cos and sin).  Timed in graphs
  // with 32 / 8, 40 / 8, 64 / 8, 16 / 2, 8 / 1 and 5 / 1 heads; us with one and with four rows, 32 / 8 heads, norm and
  // 128 channels turned: 6144 rows 2.4 and 3.5, 14,448 (301 tokens) 3.9 and 4.1, 16,384 4.15 both, 20,480 4.4 and 4.6,
  // 28,800 5.6 and 5.4, 786,432 135 and 85 (101 with two).  Without a norm, 64 turned, four are ahead from 14,448 on
  // (3.6 and 3.3); with 8 / 1 or 5 / 1 heads, whose last four are not all there, the two draw level at about 57,600
  // (20,480: 4.5 and 5.0).
  const int64_t rows = tokens * (a.Hq + 2 * num_kv_heads);
  return rows <= 16384 ? launch_append_rows<1>(a, stream) : launch_append_rows<4>(a, stream);
}

}  // namespace nv4
