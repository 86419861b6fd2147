// The 4-bit KV cache of the end-to-end model: the q/k RMSNorm + rotary + store
// that writes it and the decode attention that reads it.
//
// Format.  head_dim 128, pages of 256 tokens; for K and for V
//   codes  uint8 [pages, Hkv, 256, 64]  two 4-bit codes a byte
//   scales bf16  [pages, Hkv, 256, 4]   one per 32 channels
// so that a (page, KV head) tile is contiguous.  Of a group's absolute maximum a
// the scale is s = bf16(a / 7) (1 when the group is zero, at least the BF16
// tiny; NaN when a value of the group is not finite, so that the group reads
// back as NaN); the code of x is c = round-half-even(x / s) clamped to [-7, 7],
// held as c + 8.  72 bytes per token, KV head and side instead of BF16's 256.
//
// Four consecutive channels of a token make a 16-bit unit, the lowest channel
// in the lowest nibble.  The units of a row are ordered for the decode
// kernel's mma.sync fragments; with g = channel / 32 and r = channel % 32:
//   K: byte (r / 8) * 16 + g * 4 + (r % 8) / 4 * 2 of the token's 64 bytes;
//   V: byte ((r / 4) ^ (2 * (pair % 4))) * 16 + g * 4 + (t % 2) * 2 of the 128
//      bytes of the token pair t / 2.
#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kKv4D = 128;
constexpr int kKv4Page = 256;
constexpr int kKv4RowBytes = 64;    // codes of a token
constexpr int kKv4Groups = 4;       // scales of a token
constexpr int kKv4MaxGroup = 8;     // query heads per KV head

// Byte of the unit of channels 4 * lane .. 4 * lane + 3 within a token's K row.
__device__ __forceinline__ int kv4_k_unit(int lane) {
  return ((lane & 7) >> 1) * 16 + (lane >> 3) * 4 + (lane & 1) * 2;
}
// Byte of that unit of token t within its (page, head) tile of V codes.
__device__ __forceinline__ int kv4_v_unit(int t, int lane) {
  const int pair = t >> 1;
  return pair * 128 + ((lane & 7) ^ (2 * (pair & 3))) * 16 + (lane >> 3) * 4 + (t & 1) * 2;
}

// ------------------------------------------------------------ store
// One warp per (token, head) of the fused QKV output, four channels a lane.
// K is normalised and rotated in 64 bits and rounded once to FP32 before it is
// quantised: a code depends on which side of a border x / s lies, and with
// FP32 sums it would depend on the order of the sum.  x / s itself is an IEEE
// FP32 quotient: for a 24-bit x and an 8-bit s it never rounds onto a
// half-integer that the exact quotient does not hit, so the code is the exact
// quotient's.  q needs no such care: FP32, rounded once to BF16.
struct Kv4StoreArgs {
  const uint16_t* qkv;
  const uint16_t* q_weight;
  const uint16_t* k_weight;
  const float* cos_sin;
  const int64_t* positions;
  const int* slot_mapping;
  uint16_t* q_out;
  uint16_t* k_out;  // values held by the cache, or nullptr
  uint16_t* v_out;
  uint8_t* k_codes;
  uint16_t* k_scales;
  uint8_t* v_codes;
  uint16_t* v_scales;
  int64_t max_position, num_slots;
  double eps;
  int T, Hq, Hkv;
};

// Quantises a lane's four values with its group (8 lanes): the unit of codes
// and the group's scale.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&x)[4], uint16_t& scale_bits, float (&value)[4]) {
  uint32_t top = 0;  // as bits: an infinity or NaN is above every number
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int m = 1; m <= 4; m <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
  float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__uint_as_float(top), 7.0f)));
  s = fmaxf(s, kBf16Tiny);
  if (top == 0) s = 1.0f;
  if (top >= 0x7F800000u) s = __uint_as_float(0x7FC00000u);
  scale_bits = static_cast<uint16_t>(__float_as_uint(s) >> 16);
  uint32_t unit = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -7.0f), 7.0f);
    unit |= static_cast<uint32_t>(static_cast<int>(c) + 8) << (4 * i);
    value[i] = c * s;
  }
  return unit;
}

__global__ void __launch_bounds__(256) qk_norm_rope_store_kv4_kernel(const Kv4StoreArgs p) {
  const int heads = p.Hq + 2 * p.Hkv;
  const int64_t gw = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (gw >= static_cast<int64_t>(p.T) * heads) return;
  const int t = static_cast<int>(gw / heads), h = static_cast<int>(gw - static_cast<int64_t>(t) * heads);
  const uint2 raw = *reinterpret_cast<const uint2*>(p.qkv + gw * kKv4D + lane * 4);
  const float x[4] = {bf16lo_to_f32(raw.x), bf16hi_to_f32(raw.x), bf16lo_to_f32(raw.y), bf16hi_to_f32(raw.y)};

  float y[4];
  if (h < p.Hq + p.Hkv) {
    const uint2 wr = *reinterpret_cast<const uint2*>((h < p.Hq ? p.q_weight : p.k_weight) + lane * 4);
    const float w[4] = {bf16lo_to_f32(wr.x), bf16hi_to_f32(wr.x), bf16lo_to_f32(wr.y), bf16hi_to_f32(wr.y)};
    const int64_t pos = p.positions[t];
    float4 c4 = make_float4(NAN, NAN, NAN, NAN), s4 = c4;  // a position beyond the table: NaN, and an error
    if (pos >= 0 && pos < p.max_position) {
      const float* cs = p.cos_sin + pos * kKv4D + (lane & 15) * 4;
      c4 = *reinterpret_cast<const float4*>(cs);
      s4 = *reinterpret_cast<const float4*>(cs + kKv4D / 2);
    } else if (lane == 0) {
      record_error(kErrBadPosition);
    }
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
    if (h < p.Hq) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
      const float r = rsqrtf(ss * (1.0f / kKv4D) + static_cast<float>(p.eps));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float n = x[i] * r * w[i];
        const float o = __shfl_xor_sync(0xffffffffu, n, 16);
        y[i] = lane < 16 ? n * c[i] - o * s[i] : n * c[i] + o * s[i];
      }
    } else {
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += static_cast<double>(x[i] * x[i]);  // 16 significant bits: exact in FP32
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
      const double r = rsqrt(ss * (1.0 / kKv4D) + p.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double n = static_cast<double>(x[i]) * r * static_cast<double>(w[i]);
        const double o = __shfl_xor_sync(0xffffffffu, n, 16);
        const double cd = c[i], sd = s[i];
        y[i] = static_cast<float>(lane < 16 ? n * cd - o * sd : n * cd + o * sd);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = x[i];
  }
  if (h < p.Hq) {
    *reinterpret_cast<uint2*>(p.q_out + (static_cast<int64_t>(t) * p.Hq + h) * kKv4D + lane * 4) =
        make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    return;
  }
  const bool is_k = h < p.Hq + p.Hkv;
  const int kvh = is_k ? h - p.Hq : h - p.Hq - p.Hkv;
  uint16_t scale;
  float value[4];
  const uint32_t unit = kv4_quantise(y, scale, value);
  uint16_t* values = is_k ? p.k_out : p.v_out;
  if (values != nullptr)
    *reinterpret_cast<uint2*>(values + (static_cast<int64_t>(t) * p.Hkv + kvh) * kKv4D + lane * 4) =
        make_uint2(pack_bf16x2(value[0], value[1]), pack_bf16x2(value[2], value[3]));
  const int slot = p.slot_mapping != nullptr ? p.slot_mapping[t] : -1;
  if (slot < 0) return;
  if (slot >= p.num_slots) {
    if (lane == 0) record_error(kErrBadSlot);
    return;
  }
  const int row = slot % kKv4Page;
  const int64_t tile = static_cast<int64_t>(slot / kKv4Page) * p.Hkv + kvh;
  uint8_t* codes = (is_k ? p.k_codes : p.v_codes) + tile * (kKv4Page * kKv4RowBytes);
  uint16_t* scales = (is_k ? p.k_scales : p.v_scales) + (tile * kKv4Page + row) * kKv4Groups;
  const int at = is_k ? row * kKv4RowBytes + kv4_k_unit(lane) : kv4_v_unit(row, lane);
  *reinterpret_cast<uint16_t*>(codes + at) = static_cast<uint16_t>(unit);
  if ((lane & 7) == 0) scales[lane >> 3] = scale;
}

int launch_qk_norm_rope_store_kv4(const void* qkv, const void* q_weight, const void* k_weight, const float* cos_sin,
                                  const int64_t* positions, const int* slot_mapping, void* q_out, void* k_out,
                                  void* v_out, void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                                  int64_t tokens, int64_t num_heads, int64_t num_kv_heads, int64_t num_pages,
                                  int64_t max_position, double eps, cudaStream_t stream) {
  Kv4StoreArgs a;
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.q_weight = static_cast<const uint16_t*>(q_weight);
  a.k_weight = static_cast<const uint16_t*>(k_weight);
  a.cos_sin = cos_sin;
  a.positions = positions;
  a.slot_mapping = slot_mapping;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  a.v_out = static_cast<uint16_t*>(v_out);
  a.k_codes = static_cast<uint8_t*>(k_codes);
  a.k_scales = static_cast<uint16_t*>(k_scales);
  a.v_codes = static_cast<uint8_t*>(v_codes);
  a.v_scales = static_cast<uint16_t*>(v_scales);
  a.max_position = max_position;
  a.num_slots = num_pages * kKv4Page;
  a.eps = eps;
  a.T = static_cast<int>(tokens);
  a.Hq = static_cast<int>(num_heads);
  a.Hkv = static_cast<int>(num_kv_heads);
  const int64_t warps = tokens * (num_heads + 2 * num_kv_heads);
  return launch_kernel(qk_norm_rope_store_kv4_kernel, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(256), 0,
                       stream, false, a);
}

// ------------------------------------------------------------ decode attention
// One CTA per (page of the context, KV head, sequence), a warp per token: a
// lane holds four channels of q for every query head of the group, the dot
// products are summed over the warp, and each warp keeps its own running
// maximum, sum and output, merged at the end of the page into a partial that a
// second kernel joins.
struct Kv4AttnArgs {
  const uint16_t* q;  // [B, Hq, 128]
  const uint8_t* k_codes;
  const uint16_t* k_scales;
  const uint8_t* v_codes;
  const uint16_t* v_scales;
  const int* block_tables;  // [B, max_pages]
  const int* context_lens;
  float* o_part;   // [B, Hq, max_pages, 128]
  float* ml_part;  // [B, Hq, max_pages, 2]
  int64_t num_pages;
  int Hq, Hkv, max_pages;
  float scale_log2;
};

__global__ void __launch_bounds__(128) paged_decode_attention_kv4_kernel(const Kv4AttnArgs p) {
  __shared__ float red[4][kKv4MaxGroup][kKv4D];
  __shared__ float ml[4][kKv4MaxGroup][2];
  const int pi = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int ctx = p.context_lens[b];
  if (pi * kKv4Page >= ctx) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv;
  int ntok = min(kKv4Page, ctx - pi * kKv4Page);
  const int page = p.block_tables[static_cast<int64_t>(b) * p.max_pages + pi];
  if (page < 0 || page >= p.num_pages) {  // its tokens count as absent
    if (threadIdx.x == 0) record_error(kErrBadPage);
    ntok = 0;
  }
  const int64_t tile = static_cast<int64_t>(page) * p.Hkv + kvh;
  const uint8_t* kc = p.k_codes + tile * (kKv4Page * kKv4RowBytes);
  const uint8_t* vc = p.v_codes + tile * (kKv4Page * kKv4RowBytes);
  const uint16_t* ks = p.k_scales + tile * (kKv4Page * kKv4Groups);
  const uint16_t* vs = p.v_scales + tile * (kKv4Page * kKv4Groups);
  float q[kKv4MaxGroup][4], o[kKv4MaxGroup][4], m[kKv4MaxGroup], l[kKv4MaxGroup];
#pragma unroll
  for (int h = 0; h < kKv4MaxGroup; ++h) {
    m[h] = -1e30f;
    l[h] = 0.0f;
    const uint2 raw = h < G ? *reinterpret_cast<const uint2*>(
                                  p.q + (static_cast<int64_t>(b) * p.Hq + kvh * G + h) * kKv4D + lane * 4)
                            : make_uint2(0, 0);
    q[h][0] = bf16lo_to_f32(raw.x), q[h][1] = bf16hi_to_f32(raw.x);
    q[h][2] = bf16lo_to_f32(raw.y), q[h][3] = bf16hi_to_f32(raw.y);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[h][i] = 0.0f;
  }
  for (int t = warp; t < ntok; t += 4) {
    const uint32_t ku = *reinterpret_cast<const uint16_t*>(kc + t * kKv4RowBytes + kv4_k_unit(lane));
    const uint32_t vu = *reinterpret_cast<const uint16_t*>(vc + kv4_v_unit(t, lane));
    const float ksc = bf16_bits_to_f32(ks[t * kKv4Groups + (lane >> 3)]);
    const float vsc = bf16_bits_to_f32(vs[t * kKv4Groups + (lane >> 3)]);
    float k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = ksc * static_cast<float>(static_cast<int>((ku >> (4 * i)) & 15) - 8);
      v[i] = vsc * static_cast<float>(static_cast<int>((vu >> (4 * i)) & 15) - 8);
    }
#pragma unroll
    for (int h = 0; h < kKv4MaxGroup; ++h) {
      if (h >= G) break;
      float s = q[h][0] * k[0] + q[h][1] * k[1] + q[h][2] * k[2] + q[h][3] * k[3];
#pragma unroll
      for (int x = 16; x >= 1; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= p.scale_log2;
      const float mn = fmaxf(m[h], s), alpha = exp2f(m[h] - mn), e = exp2f(s - mn);
      m[h] = mn;
      l[h] = l[h] * alpha + e;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[h][i] = o[h][i] * alpha + e * v[i];
    }
  }
#pragma unroll
  for (int h = 0; h < kKv4MaxGroup; ++h) {
    if (h >= G) break;
    *reinterpret_cast<float4*>(&red[warp][h][lane * 4]) = make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
    if (lane == 0) ml[warp][h][0] = m[h], ml[warp][h][1] = l[h];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * kKv4D; i += 128) {
    const int h = i / kKv4D, d = i % kKv4D;
    float M = -1e30f, L = 0.0f, acc = 0.0f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w][h][0]);
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(ml[w][h][0] - M);
      acc += f * red[w][h][d];
      L += f * ml[w][h][1];
    }
    const int64_t part = (static_cast<int64_t>(b) * p.Hq + kvh * G + h) * p.max_pages + pi;
    p.o_part[part * kKv4D + d] = acc;
    if (d == 0) p.ml_part[part * 2] = M, p.ml_part[part * 2 + 1] = L;
  }
}

__global__ void __launch_bounds__(128) kv4_merge_kernel(const Kv4AttnArgs p, uint16_t* __restrict__ out) {
  const int64_t bh = blockIdx.x;
  const int b = static_cast<int>(bh / p.Hq), d = threadIdx.x;
  const int np = min(p.max_pages, (max(p.context_lens[b], 0) + kKv4Page - 1) / kKv4Page);
  const int64_t base = bh * p.max_pages;
  float M = -1e30f, L = 0.0f, acc = 0.0f;
  for (int i = 0; i < np; ++i) M = fmaxf(M, p.ml_part[(base + i) * 2]);
  for (int i = 0; i < np; ++i) {
    const float f = exp2f(p.ml_part[(base + i) * 2] - M);
    acc += f * p.o_part[(base + i) * kKv4D + d];
    L += f * p.ml_part[(base + i) * 2 + 1];
  }
  out[bh * kKv4D + d] = __bfloat16_as_ushort(__float2bfloat16_rn(L == 0.0f ? 0.0f : acc / L));
}

int64_t paged_attention_kv4_workspace_bytes(int64_t batch, int64_t num_heads, int64_t max_pages) {
  return batch * num_heads * max_pages * (kKv4D + 2) * 4;
}

int launch_paged_decode_attention_kv4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                      const void* v_scales, const int* block_tables, const int* context_lens,
                                      void* out, void* workspace, int64_t batch, int64_t num_heads,
                                      int64_t num_kv_heads, int64_t num_pages, int64_t max_pages, float scale,
                                      cudaStream_t stream) {
  Kv4AttnArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k_codes = static_cast<const uint8_t*>(k_codes);
  a.k_scales = static_cast<const uint16_t*>(k_scales);
  a.v_codes = static_cast<const uint8_t*>(v_codes);
  a.v_scales = static_cast<const uint16_t*>(v_scales);
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.o_part = static_cast<float*>(workspace);
  a.ml_part = a.o_part + batch * num_heads * max_pages * kKv4D;
  a.num_pages = num_pages;
  a.Hq = static_cast<int>(num_heads);
  a.Hkv = static_cast<int>(num_kv_heads);
  a.max_pages = static_cast<int>(max_pages);
  a.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid(static_cast<unsigned>(max_pages), static_cast<unsigned>(num_kv_heads),
                  static_cast<unsigned>(batch));
  const int rc = launch_kernel(paged_decode_attention_kv4_kernel, grid, dim3(128), 0, stream, false, a);
  if (rc != NV4_OK) return rc;
  return launch_kernel(kv4_merge_kernel, dim3(static_cast<unsigned>(batch * num_heads)), dim3(kKv4D), 0, stream,
                       false, a, static_cast<uint16_t*>(out));
}

}  // namespace nv4
