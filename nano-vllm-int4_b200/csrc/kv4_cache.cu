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
#include <numeric>

#include "nv4_device.cuh"
#include "nv4_launch.h"

namespace nv4 {

constexpr int kKv4D = 128;
constexpr int kKv4Page = 256;
constexpr int kKv4RowBytes = 64;    // codes of a token
constexpr int kKv4Groups = 4;       // scales of a token
constexpr int kKv4MaxGroup = 8;     // query heads per KV head

// ------------------------------------------------------------ store
// Eight lanes per row ((token, head) of the fused QKV output), 16 channels a lane:
// eight and the eight that the rotation pairs them with (with half as many a
// lane, what every row costs besides its values made it 1.4 times slower).  The
// octets of a full grid walk the rows; their number is coprime to the heads, so
// that each takes q, K and V rows in turn (a K row costs four times a q row).
// The next row is on its way meanwhile.  Bound by HBM for long prompts: a row is
// read and written once.
//
// A K code depends on which side of a border x / s lies, and with FP32 sums that
// would depend on the order of the sum.  So K is computed beyond FP32 and rounded
// once to it: the sum of squares and its root in 64 bits, norm weight and
// rotation as unevaluated sums of two FP32 numbers (k = r (P c -+ P' s) with P = x w
// exact; about 2^-46 off before the rounding).  That is 18 FP32 operations a
// value; in FP64 the conversions alone took twice the time.  q needs no such
// care: FP32, rounded once to BF16.
//
// Measured (32 / 8 heads, with the values): 16384 tokens 103 us = 4.1 TB/s (0.63 of
// the measured copy rate), 301 tokens of 40 / 8 heads 4.8 us, 32 tokens 3.5 us.
// Next: the latency of cos, sin and the weights, which every row loads again, and the
// two-term arithmetic, which every K value takes though only those next to a border
// need it; no pipe is full (0.60 instructions a cycle and scheduler).  Tried and not
// better: a ring of four rows in shared memory, cos and sin before the row, 64-thread
// CTAs, five, seven or eight CTAs an SM.
struct Kv4StoreArgs {
  const uint16_t* qkv;
  const uint16_t* q_weight;
  const uint16_t* k_weight;
  const float* cos_sin;
  const int64_t* positions;
  const int* slot_mapping;
  uint16_t* q_out;
  uint16_t* k_out;  // values held by the cache, rounded to BF16, or nullptr
  uint16_t* v_out;
  uint8_t* k_codes;
  uint16_t* k_scales;
  uint8_t* v_codes;
  uint16_t* v_scales;
  int64_t max_position, num_slots;
  double eps;
  int T, Hq, Hkv;
  int walkers;                  // octets that walk the rows, each by as many rows
  int walk_tokens, walk_heads;  // that many rows, as tokens and heads
};

// A lane's channels 8 l .. 8 l + 7 and 64 on, of the 8 lanes of a row.
constexpr int kKv4RowLanes = 8;
struct RowPart {
  uint4 lo, hi;
};
__device__ __forceinline__ RowPart load_row(const uint16_t* row, int lane) {
  const uint4* p = reinterpret_cast<const uint4*>(row) + lane;
  return {__ldg(p), __ldg(p + 8)};
}
// The lane's values as pairs of FP32: channels (0, 1), ..., (6, 7), then 64 on.
__device__ __forceinline__ void unpack_row(const RowPart& r, uint64_t (&x)[8]) {
  const uint32_t w[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = pair(bf16lo_to_f32(w[i]), bf16hi_to_f32(w[i]));
}
__device__ __forceinline__ uint32_t pack_pair(uint64_t x) {
  float lo, hi;
  unpair(x, lo, hi);
  return pack_bf16x2(lo, hi);
}
__device__ __forceinline__ void store_row(uint16_t* row, int lane, const uint64_t (&x)[8]) {
  uint4* p = reinterpret_cast<uint4*>(row) + lane;
  __stcs(p, make_uint4(pack_pair(x[0]), pack_pair(x[1]), pack_pair(x[2]), pack_pair(x[3])));
  __stcs(p + 8, make_uint4(pack_pair(x[4]), pack_pair(x[5]), pack_pair(x[6]), pack_pair(x[7])));
}

// RMSNorm and rotary embedding over the lanes of `mask`; c, s: cos and sin of the
// lane's eight channels.
__device__ __forceinline__ void norm_rope_q(uint64_t (&x)[8], const uint64_t (&w)[8], const uint64_t (&c)[4],
                                            const uint64_t (&s)[4], float eps, uint32_t mask) {
  uint64_t s2 = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) s2 = fma2(x[i], x[i], s2);
  float ss, other;
  unpair(s2, ss, other);
  ss += other;
#pragma unroll
  for (int m = kKv4RowLanes / 2; m >= 1; m >>= 1) ss += __shfl_xor_sync(mask, ss, m);
  const float r = rsqrtf(ss * (1.0f / kKv4D) + eps);
  const uint64_t rr = pair(r, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t a = mul2(mul2(x[i], rr), w[i]), b = mul2(mul2(x[i + 4], rr), w[i + 4]);
    x[i] = sub2(mul2(a, c[i]), mul2(b, s[i]));
    x[i + 4] = fma2(b, c[i], mul2(a, s[i]));
  }
}
// r (a c + b s) of exact a, b, with r = rh + rl: both products and their sum with
// what rounding takes from them.
__device__ __forceinline__ uint64_t turn_k(uint64_t a, uint64_t b, uint64_t c, uint64_t s, uint64_t rh, uint64_t rl) {
  const uint64_t ac = mul2(a, c), bs = mul2(b, s);
  const uint64_t low = add2(fma2(a, c, sub2(0, ac)), fma2(b, s, sub2(0, bs)));
  const uint64_t sum = add2(ac, bs), z = sub2(sum, ac);
  const uint64_t rest = add2(add2(sub2(ac, sub2(sum, z)), sub2(bs, z)), low);
  const uint64_t y = mul2(sum, rh);
  return add2(y, fma2(rest, rh, fma2(sum, rl, fma2(sum, rh, sub2(0, y)))));
}
__device__ __forceinline__ void norm_rope_k(uint64_t (&x)[8], const uint64_t (&w)[8], const uint64_t (&c)[4],
                                            const uint64_t (&s)[4], double eps, uint32_t mask) {
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float lo, hi;
    unpair(x[i], lo, hi);
    ss = fma(static_cast<double>(lo), static_cast<double>(lo), ss);
    ss = fma(static_cast<double>(hi), static_cast<double>(hi), ss);
  }
#pragma unroll
  for (int m = kKv4RowLanes / 2; m >= 1; m >>= 1) ss += __shfl_xor_sync(mask, ss, m);
  const double r = rsqrt(ss * (1.0 / kKv4D) + eps);
  const float h = static_cast<float>(r), l = static_cast<float>(r - static_cast<double>(h));
  const uint64_t rh = pair(h, h), rl = pair(l, l);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t a = mul2(x[i], w[i]), b = mul2(x[i + 4], w[i + 4]);  // 16 significant bits: exact
    x[i] = turn_k(a, sub2(0, b), c[i], s[i], rh, rl);
    x[i + 4] = turn_k(b, a, c[i], s[i], rh, rl);
  }
}

// Quantises eight values of a lane with their group (four lanes): the codes, a
// nibble a channel, and the scale; x becomes the values that the codes stand for.
__device__ __forceinline__ uint32_t kv4_quantise(uint64_t* x, float& scale, uint32_t mask) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpair(x[i], v[2 * i], v[2 * i + 1]);
  uint32_t top = 0;  // as bits: an infinity or NaN is above every number
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(mask, top, 1));
  top = max(top, __shfl_xor_sync(mask, top, 2));
  scale = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__uint_as_float(top), 7.0f)));
  scale = fmaxf(scale, kBf16Tiny);
  if (top == 0) scale = 1.0f;
  if (top >= 0x7F800000u) scale = __uint_as_float(0x7FC00000u);
  // x / s to the last bit or next to it: q + (x - q s) / s, the remainder exact.
  // That rounds to the exact quotient's integer: s has 8 significant bits, so a
  // quotient off a half-integer h is off by more than 2^-24 (1 + 2^-8) h, above
  // half a unit of h by 2^-33 h, and the error is 2^-47 h; h itself comes out
  // exactly.  Below 2^-80 the remainder would underflow: an IEEE division.
  const float inv = __frcp_rn(scale);
  const uint64_t ii = pair(inv, inv), minus = pair(-scale, -scale);
  if (scale >= 0x1p-80f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t q = mul2(x[i], ii);
      unpair(fma2(fma2(q, minus, x[i]), ii, q), v[2 * i], v[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fdiv_rn(v[i], scale);
  }
  // Rounded to even in the last place of 1.5 * 2^23, whose low 22 bits are 0; + 8
  // makes the nibble.
  uint32_t low = 0, high = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    v[i] = fminf(fmaxf(v[i], -7.0f), 7.0f) + 12582920.0f;
    v[i + 4] = fminf(fmaxf(v[i + 4], -7.0f), 7.0f) + 12582920.0f;
    low = low * 16 + __float_as_uint(v[i]);
    high = high * 16 + __float_as_uint(v[i + 4]);
  }
  const uint64_t ss = pair(scale, scale), magic = pair(12582920.0f, 12582920.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = mul2(sub2(pair(v[2 * i], v[2 * i + 1]), magic), ss);
  return __byte_perm(low, high, 0x5410);
}

constexpr int kKv4StoreThreads = 128, kKv4StoreCtas = 6;  // an SM
__global__ void __launch_bounds__(kKv4StoreThreads, kKv4StoreCtas)
    qk_norm_rope_store_kv4_kernel(const Kv4StoreArgs p) {
  const int heads = p.Hq + 2 * p.Hkv, lane = threadIdx.x & 7;
  const uint32_t mask = 0xFFu << (threadIdx.x & 24);  // the octets go their own ways
  const int first = blockIdx.x * (kKv4StoreThreads / kKv4RowLanes) + (threadIdx.x >> 3);
  int t = first / heads, h = first - t * heads;
  if (first >= p.walkers || t >= p.T) return;
  const uint16_t* src = p.qkv + static_cast<int64_t>(first) * kKv4D;
  const int64_t stride = static_cast<int64_t>(p.walkers) * kKv4D;
  RowPart raw = load_row(src, lane);
  int64_t pos = p.positions[t];
  while (true) {
    uint64_t x[8];
    unpack_row(raw, x);
    const int row_t = t, row_h = h;
    const int64_t row_pos = pos;
    t += p.walk_tokens, h += p.walk_heads;  // the row after this one
    if (h >= heads) h -= heads, ++t;
    const bool more = t < p.T;
    if (more) {
      src += stride;
      raw = load_row(src, lane);
      pos = p.positions[t];
    }
    const bool is_q = row_h < p.Hq, is_k = !is_q && row_h < p.Hq + p.Hkv;
    if (is_q || is_k) {
      uint64_t w[8], c[4], s[4];
      unpack_row(load_row(is_q ? p.q_weight : p.k_weight, lane), w);
      if (static_cast<uint64_t>(row_pos) < static_cast<uint64_t>(p.max_position)) {
        const ulonglong2* cs = reinterpret_cast<const ulonglong2*>(p.cos_sin + row_pos * kKv4D) + lane * 2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const ulonglong2 cc = __ldg(cs + i), sn = __ldg(cs + 16 + i);
          c[2 * i] = cc.x, c[2 * i + 1] = cc.y, s[2 * i] = sn.x, s[2 * i + 1] = sn.y;
        }
      } else {  // beyond the table: NaN, and an error
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = s[i] = pair(NAN, NAN);
        if (lane == 0) record_index_error(kErrBadPosition);
      }
      if (is_q) norm_rope_q(x, w, c, s, static_cast<float>(p.eps), mask);
      else norm_rope_k(x, w, c, s, p.eps, mask);
    }
    if (is_q) {
      store_row(p.q_out + (static_cast<int64_t>(row_t) * p.Hq + row_h) * kKv4D, lane, x);
    } else {
      const int kvh = row_h - (is_k ? p.Hq : p.Hq + p.Hkv);
      float scale[2];
      uint32_t word[2];  // of groups lane / 4 and 2 + lane / 4
#pragma unroll
      for (int i = 0; i < 2; ++i) word[i] = kv4_quantise(x + 4 * i, scale[i], mask);
      uint16_t* values = is_k ? p.k_out : p.v_out;
      if (values != nullptr) store_row(values + (static_cast<int64_t>(row_t) * p.Hkv + kvh) * kKv4D, lane, x);
      const int slot = p.slot_mapping != nullptr ? p.slot_mapping[row_t] : -1;
      if (slot >= 0 && slot < p.num_slots) {
        const int token = slot % kKv4Page, g = lane >> 2, run = lane & 3;
        const int64_t tile = static_cast<int64_t>(slot / kKv4Page) * p.Hkv + kvh;
        if (is_k) {
          uint8_t* codes = p.k_codes + (tile * kKv4Page + token) * kKv4RowBytes + run * 16 + g * 4;
          *reinterpret_cast<uint32_t*>(codes) = word[0];
          *reinterpret_cast<uint32_t*>(codes + 8) = word[1];
        } else {
          uint8_t* codes = p.v_codes + tile * (kKv4Page * kKv4RowBytes) + (token >> 1) * 128 + g * 4 + (token & 1) * 2;
          const int turn = 2 * ((token >> 1) & 3);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint8_t* at = codes + ((2 * run + i) ^ turn) * 16;
            *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(word[0] >> (16 * i));
            *reinterpret_cast<uint16_t*>(at + 8) = static_cast<uint16_t>(word[1] >> (16 * i));
          }
        }
        if (run == 0) {
          uint16_t* scales = (is_k ? p.k_scales : p.v_scales) + (tile * kKv4Page + token) * kKv4Groups + g;
          scales[0] = static_cast<uint16_t>(__float_as_uint(scale[0]) >> 16);
          scales[2] = static_cast<uint16_t>(__float_as_uint(scale[1]) >> 16);
        }
      } else if (slot >= 0 && lane == 0) {
        record_index_error(kErrBadSlot);
      }
    }
    if (!more) return;
  }
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
  // as many CTAs as run at once, or as there are rows for
  constexpr int64_t kRows = kKv4StoreThreads / kKv4RowLanes;
  const int64_t heads = num_heads + 2 * num_kv_heads, rows = tokens * heads;
  const int64_t ctas =
      std::min<int64_t>((rows + kRows - 1) / kRows, kKv4StoreCtas * static_cast<int64_t>(device_sm_count()));
  int64_t walkers = ctas * kRows;
  if (rows > walkers)
    while (walkers > 1 && std::gcd(walkers, heads) != 1) --walkers;
  a.walkers = static_cast<int>(walkers);
  a.walk_tokens = static_cast<int>(walkers / heads);
  a.walk_heads = static_cast<int>(walkers % heads);
  return launch_kernel(qk_norm_rope_store_kv4_kernel, dim3(static_cast<unsigned>(ctas)),
                       dim3(kKv4StoreThreads), 0, stream, false, a);
}

// ------------------------------------------------------------ decode attention
// o[h] = sum_t softmax_t(scale q[h].k_t) v_t over a sequence's tokens, for the G
// query heads that share a KV head.  Per token and KV head 144 bytes are read
// and 256 codes widened; at HBM rate an SM has about 6 cycles for that, so the
// work per code is what the kernel is arranged around.
//
// Split: the tokens of all (sequence, KV head) jobs form one line of 128-token
// units, cut evenly over a fixed grid (four CTAs an SM), so ragged lengths cost
// nothing.  The lengths live on the device: every CTA makes the prefix sum
// itself.  A job that lies within one CTA is finished there; else each CTA
// writes an unnormalised partial to the workspace (two slots a CTA: the job
// that it continues, the job that it leaves) and a second kernel joins them in
// order.  Units come through a ring by bulk copies (a unit of a page is
// contiguous); four warps take 16 tokens at a time.  One thread of them issues the
// copies: a warp of its own for that would hold a fifth of the registers.
//
// Arithmetic, per 16 tokens and warp, on mma.sync:
//   S^T [16 tokens x 8 heads], m16n8k16 in BF16: A = K codes as 128 + u (the nibble
//     u = c + 8 in the low mantissa bits of 128: one mask-and-or), B = q. The
//     excess of 136 leaves through the accumulator's start, -136 sum(q), so K needs no
//     subtraction. The scale is one per token and 32 channels: two MMAs, one FMA.
//   O^T [128 channels x 8 heads], likewise: A = V codes, exactly (accumulated over
//     the whole context, so the excess is subtracted first), B = p * scale in two
//     BF16 terms, whose products go into the same accumulators: the output's own
//     rounding is then the only one that shows (0.0017 of the norm; 0.0023 with one
//     term, which takes 102 us instead of 114 for 64 ragged sequences, and nothing less
//     for a single short one).
// p reaches its B fragment with movmatrix.  The running maximum is moved only
// when a score exceeds it by 2^8 (p and its sum are at most 2^8 larger then).
//
// Measured (32 / 8 heads, with the merge): 32 x 4.2k tokens 56 us = 2.8 TB/s, 64
// ragged up to 16k 114 us = 3.1 TB/s (0.48 of the measured copy rate), one of 700
// tokens 7.9 us.  Bound by the latency of a warp's own chain (load, widen, two MMAs
// a group, FMAs, vote, exponential, pack, movmatrix, MMA) with four warps a
// scheduler: 0.57 instructions a cycle and scheduler, the ALU at half of its rate, the
// tensor pipe at 25%, HBM at 0.43, none of them full.  With one term of the
// probabilities (101 us for the ragged case) the copies took 65 us without the
// products and the products 99 without the copies; 64 mask-and-or instructions fewer
// of about 303 per 16 tokens gave 15%.  Tried then and slower (64 ragged): units of 64
// tokens, five CTAs an SM at 96 registers (110 us), a warp of its own for the copies
// (105), two tiles of a warp at once, eight-warp CTAs; K as 8-bit integers against q
// in 16-bit fixed point lost precision at large scores.
constexpr int kKv4Warps = 4;
constexpr int kKv4Threads = kKv4Warps * 32;
constexpr int kKv4Tiles = 2;                          // 16-token tiles a warp takes of a unit
constexpr int kKv4Unit = kKv4Warps * kKv4Tiles * 16;  // tokens of a unit; divides the page
constexpr int kKv4Stages = 2;  // what four CTAs an SM leave room for
constexpr int kKv4CodeBytes = kKv4Unit * kKv4RowBytes;       // of K or V, a unit
constexpr int kKv4ScaleBytes = kKv4Unit * kKv4Groups * 2;
constexpr int kKv4RedStride = kKv4D + 4;  // floats; conflict-free stores of the fragments
constexpr int kKv4CtasPerSm = 4;
constexpr int kKv4MaxCtas = kKv4CtasPerSm * 160;
constexpr int kKv4SlotFloats = kKv4MaxGroup * (kKv4D + 2);  // a partial: outputs, then (max, sum) per head
constexpr float kKv4NoMax = -3.4028234e38f;  // the lowest FP32: any finite score is above it or equal
constexpr float kKv4Slack = 8.0f;  // log2 units by which a score may pass the running maximum

// Shared memory: the stages (K, V, K scales, V scales, q), then the warps' outputs
// of four heads at a time.
constexpr int kKv4QAt = 2 * kKv4CodeBytes + 2 * kKv4ScaleBytes;
constexpr int kKv4StageBytes = kKv4QAt + kKv4MaxGroup * kKv4D * 2;
constexpr int kKv4RedAt = kKv4Stages * kKv4StageBytes;
constexpr int kKv4Smem = kKv4RedAt + kKv4Warps * 4 * kKv4RedStride * 4;

struct Kv4AttnArgs {
  const uint16_t* q;  // [B, Hq, 128]
  const uint8_t* k_codes;
  const uint16_t* k_scales;
  const uint8_t* v_codes;
  const uint16_t* v_scales;
  const int* block_tables;  // [B, max_pages]
  const int* context_lens;
  uint16_t* out;
  float* partials;   // [2 * CTAs][kKv4SlotFloats]
  int64_t* starts;   // [B + 1]: first unit of each sequence, per KV head
  int64_t num_pages;
  int B, Hq, Hkv, max_pages;
  float scale_log2;
};

struct Kv4Meta {  // of a unit in the ring
  int job;     // b * Hkv + h
  int tokens;  // valid tokens, 0 for an absent page
  int first;   // first unit of the job in this CTA
  int last;    // 0, or 1 + where the result goes: 1 the output, 2 / 3 partial slot 0 / 1
};

// What the thread that feeds the ring keeps between units, in shared memory so that
// it takes no registers meanwhile.
struct Kv4Feed {
  int64_t left;      // units to copy
  int64_t row;       // cache row of the next unit
  int b, h, k;       // its sequence, KV head and place among the job's n units
  int n, ctx;
  int next;          // the page of the next unit that begins one
  int first, begun;  // the unit is the job's first in this CTA; the job began in this CTA
  int there;         // its page exists
  int issued;        // units copied
};

__device__ __forceinline__ int kv4_context(const Kv4AttnArgs& p, int b) {
  return min(max(p.context_lens[b], 0), p.max_pages * kKv4Page);
}
__device__ __forceinline__ int kv4_units(int ctx) { return (ctx + kKv4Unit - 1) / kKv4Unit; }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Transpose of an 8x8 matrix of 16-bit elements held as mma fragments.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_bf16_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1, float c0, float c1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %10, %11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mma_bf16_acc(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Nibble I of both halves of w as BF16: 128 + u. magic = 0x43004300 (128, 128),
// in a register that the compiler does not know: with two constants it makes two
// logic operations of (w & mask) | magic.
template <int I>
__device__ __forceinline__ uint32_t nibbles_plus128(uint32_t w, uint32_t magic) {
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(v) : "r"(w >> (4 * I)), "r"(magic));
  return v;
}
// The same as codes: (128 + u) - 136, exact.
template <int I>
__device__ __forceinline__ uint32_t nibbles_code(uint32_t w, uint32_t magic) {
  const uint32_t v = nibbles_plus128<I>(w, magic);
  __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&v);
  x = __hsub2(x, __floats2bfloat162_rn(136.0f, 136.0f));
  return *reinterpret_cast<uint32_t*>(&x);
}

// First unit of CTA i of n over `total` units.
__device__ __forceinline__ int64_t kv4_cut(int64_t total, int i, int n) { return total * i / n; }

__global__ void __launch_bounds__(kKv4Threads, kKv4CtasPerSm) paged_decode_attention_kv4_kernel(const Kv4AttnArgs p) {
  extern __shared__ __align__(128) uint8_t smem_kv4[];
  __shared__ uint64_t full[kKv4Stages], empty[kKv4Stages], red_full, red_free;
  __shared__ Kv4Meta meta[kKv4Stages];
  __shared__ Kv4Feed feed;
  __shared__ int64_t sums[kKv4Threads / 32];
  __shared__ int64_t start_of_b;
  __shared__ int start_b;
  __shared__ uint32_t magic_word;
  __shared__ float red_ml[kKv4Warps][kKv4MaxGroup][2];
  float* red = reinterpret_cast<float*>(smem_kv4 + kKv4RedAt);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.Hq / p.Hkv;

  if (tid == 0) {
    magic_word = 0x43004300u;
    for (int i = 0; i < kKv4Stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kKv4Warps);
    }
    mbar_init(&red_full, kKv4Warps);
    mbar_init(&red_free, kKv4Warps);
    fence_mbar_init();
  }
  // Units of all sequences, and the sequence of this CTA's first unit: each
  // thread takes a run of sequences.
  const int per = (p.B + kKv4Threads - 1) / kKv4Threads;
  const int b_lo = min(tid * per, p.B), b_hi = min(b_lo + per, p.B);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += kv4_units(kv4_context(p, b));
  int64_t incl = mine;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, incl, m);
    if (lane >= m) incl += o;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int64_t total = 0, before = 0;
  for (int w = 0; w < kKv4Threads / 32; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const int ctas = static_cast<int>(min(total * p.Hkv, static_cast<int64_t>(gridDim.x)));  // a unit each at least
  const bool working = static_cast<int>(blockIdx.x) < ctas;
  const int64_t u0 = working ? kv4_cut(total * p.Hkv, blockIdx.x, ctas) : -1;
  const int64_t u1 = working ? kv4_cut(total * p.Hkv, blockIdx.x + 1, ctas) : -1;
  {
    int64_t at = before + incl - mine;
    for (int b = b_lo; b < b_hi; ++b) {
      const int n = kv4_units(kv4_context(p, b));
      if (u0 >= at * p.Hkv && u0 < (at + n) * p.Hkv) start_b = b, start_of_b = at;
      if (blockIdx.x == 0) p.starts[b] = at;
      at += n;
    }
    if (blockIdx.x == 0 && tid == 0) p.starts[p.B] = total;
  }
  __syncthreads();
  grid_dependents_launch();
  if (!working) return;

  // The copies of the next unit, by one thread once its stage is free.
  const auto feed_unit = [&]() {
    constexpr int kPerPage = kKv4Page / kKv4Unit;
    Kv4Feed f = feed;
    if (f.left == 0) return;
    const int st = f.issued % kKv4Stages;
    if (f.first || f.k % kPerPage == 0) {
      const int page = f.next;
      f.there = page >= 0 && page < p.num_pages;
      if (!f.there) record_index_error(kErrBadPage);
      f.row = (static_cast<int64_t>(page) * p.Hkv + f.h) * kKv4Page + (f.k % kPerPage) * kKv4Unit;
      // the page after it, of this job or the first of the next head's
      const int pi = f.k / kPerPage + 1;
      f.next = p.block_tables[static_cast<int64_t>(f.b) * p.max_pages + (pi * kPerPage < f.n ? pi : 0)];
    }
    const int tokens = f.there ? min(kKv4Unit, f.ctx - f.k * kKv4Unit) : 0;
    const bool ends = f.k + 1 == f.n;
    Kv4Meta mt;
    mt.job = f.b * p.Hkv + f.h;
    mt.tokens = tokens;
    mt.first = f.first;
    // the slot of a job that goes on from the CTA before is 0, as is that of one that begins with the CTA
    mt.last = f.left > 1 && !ends ? 0 : f.begun && ends ? 1 : f.begun && u1 - f.left - f.k > u0 ? 3 : 2;
    meta[st] = mt;
    const uint32_t rows = (tokens + 15) & ~15;
    const uint32_t q_bytes = f.first ? G * kKv4D * 2 : 0;
    mbar_arrive_expect_tx(&full[st], rows * (2 * kKv4RowBytes + 4 * kKv4Groups) + q_bytes);
    uint8_t* dst = smem_kv4 + st * kKv4StageBytes;
    if (f.first)
      bulk_load(dst + kKv4QAt, p.q + (static_cast<int64_t>(f.b) * p.Hq + f.h * G) * kKv4D, q_bytes, &full[st]);
    if (rows) {
      bulk_load(dst, p.k_codes + f.row * kKv4RowBytes, rows * kKv4RowBytes, &full[st]);
      bulk_load(dst + 2 * kKv4CodeBytes, p.k_scales + f.row * kKv4Groups, rows * kKv4Groups * 2, &full[st]);
      bulk_load(dst + kKv4CodeBytes, p.v_codes + f.row * kKv4RowBytes, rows * kKv4RowBytes, &full[st]);
      bulk_load(dst + 2 * kKv4CodeBytes + kKv4ScaleBytes, p.v_scales + f.row * kKv4Groups, rows * kKv4Groups * 2,
                &full[st]);
    }
    f.row += kKv4Unit;
    ++f.issued;
    --f.left;
    f.first = 0;
    if (ends) {
      f.k = 0, f.first = f.begun = 1;
      if (++f.h == p.Hkv) {
        f.h = 0;
        if (f.left > 0) {
          do {
            f.ctx = kv4_context(p, ++f.b);
            f.n = kv4_units(f.ctx);
          } while (f.n == 0);
          f.next = p.block_tables[static_cast<int64_t>(f.b) * p.max_pages];
        }
      }
    } else {
      ++f.k;
    }
    feed = f;
  };
  // The CTA's shared memory must outlive its copies: before leaving early, the
  // feeding thread waits for those on their way.
  const auto drain = [&]() {
    if (tid != 0) return;
    for (int i = max(feed.issued - kKv4Stages, 0); i < feed.issued; ++i)
      mbar_wait_drain(&full[i % kKv4Stages], (i / kKv4Stages) & 1);
  };
  if (tid == 0) {
    const int64_t rest = u0 - start_of_b * p.Hkv;  // units into the sequence
    Kv4Feed f;
    f.left = u1 - u0;
    f.row = 0;
    f.b = start_b;
    f.ctx = kv4_context(p, f.b);
    f.n = kv4_units(f.ctx);
    f.h = static_cast<int>(rest / f.n);
    f.k = static_cast<int>(rest - static_cast<int64_t>(f.h) * f.n);
    f.next = p.block_tables[static_cast<int64_t>(f.b) * p.max_pages + f.k / (kKv4Page / kKv4Unit)];
    f.first = 1;
    f.begun = f.k == 0;
    f.there = 1;
    f.issued = 0;
    feed = f;
    for (int i = 0; i < kKv4Stages; ++i) feed_unit();
  }
  __syncwarp();

  uint32_t magic;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(magic) : "r"(smem_u32(&magic_word)));
  const int gid = lane >> 2, tig = lane & 3;
  uint32_t qb[4][4];         // B fragments of q, per 32 channels
  float start[4][2];         // -136 sum of q over 32 channels, of heads 2 tig and 2 tig + 1
  float o[8][4];
  float m[2], l[2], top[2];  // running maximum (log2 units), sum, score limit of this maximum
  uint32_t merges = 0;
  int st = 0;
  uint32_t round = 0;
  for (int64_t left = u1 - u0; left > 0; --left) {
    if (!mbar_wait(&full[st], round, kErrTimeoutFull)) return drain();
    const uint8_t* buf = smem_kv4 + st * kKv4StageBytes;
    const Kv4Meta mt = meta[st];
    if (mt.first) {
      const uint16_t* qs = reinterpret_cast<const uint16_t*>(buf + kKv4QAt);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (gid < G) w = *reinterpret_cast<const uint4*>(qs + gid * kKv4D + j * 32 + tig * 8);
        qb[j][0] = __byte_perm(w.x, w.z, 0x5410);  // channels (0, 4), (1, 5), (2, 6), (3, 7)
        qb[j][1] = __byte_perm(w.x, w.z, 0x7632);
        qb[j][2] = __byte_perm(w.y, w.w, 0x5410);
        qb[j][3] = __byte_perm(w.y, w.w, 0x7632);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += bf16lo_to_f32(qb[j][i]) + bf16hi_to_f32(qb[j][i]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        start[j][0] = -136.0f * __shfl_sync(0xffffffffu, sum, 8 * tig);
        start[j][1] = -136.0f * __shfl_sync(0xffffffffu, sum, 8 * tig + 4);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x) m[x] = kKv4NoMax, l[x] = 0.0f, top[x] = kKv4NoMax;
    }
    // tiles warp, warp + 4, ...: a short unit is spread over all warps
#pragma unroll 1
    for (int t = warp * 16; t < mt.tokens; t += kKv4Warps * 16) {
      // scores of tokens t + gid (s[0], s[1]: heads 2 tig, 2 tig + 1) and t + gid + 8 (s[2], s[3])
      const uint4 ka = *reinterpret_cast<const uint4*>(buf + (t + gid) * kKv4RowBytes + tig * 16);
      const uint4 kb = *reinterpret_cast<const uint4*>(buf + (t + gid + 8) * kKv4RowBytes + tig * 16);
      const uint2 sa = *reinterpret_cast<const uint2*>(buf + 2 * kKv4CodeBytes + (t + gid) * 8);
      const uint2 sb = *reinterpret_cast<const uint2*>(buf + 2 * kKv4CodeBytes + (t + gid + 8) * 8);
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
      const float fa[4] = {bf16lo_to_f32(sa.x), bf16hi_to_f32(sa.x), bf16lo_to_f32(sa.y), bf16hi_to_f32(sa.y)};
      const float fb[4] = {bf16lo_to_f32(sb.x), bf16hi_to_f32(sb.x), bf16lo_to_f32(sb.y), bf16hi_to_f32(sb.y)};
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float acc[4];
        mma_bf16_from(acc, nibbles_plus128<0>(wa[j], magic), nibbles_plus128<0>(wb[j], magic),
                      nibbles_plus128<1>(wa[j], magic), nibbles_plus128<1>(wb[j], magic), qb[j][0], qb[j][1],
                      start[j][0], start[j][1]);
        mma_bf16_acc(acc, nibbles_plus128<2>(wa[j], magic), nibbles_plus128<2>(wb[j], magic),
                     nibbles_plus128<3>(wa[j], magic), nibbles_plus128<3>(wb[j], magic), qb[j][2], qb[j][3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(i < 2 ? fa[j] : fb[j], acc[i], s[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] *= p.scale_log2;
      uint2 ua = *reinterpret_cast<const uint2*>(buf + 2 * kKv4CodeBytes + kKv4ScaleBytes + (t + gid) * 8);
      uint2 ub = *reinterpret_cast<const uint2*>(buf + 2 * kKv4CodeBytes + kKv4ScaleBytes + (t + gid + 8) * 8);
      if (t + 16 > mt.tokens) {  // rows behind the last token hold anything: a probability of 0 does not undo a NaN
        if (t + gid >= mt.tokens) s[0] = s[1] = -INFINITY, ua = make_uint2(0, 0);
        if (t + gid + 8 >= mt.tokens) s[2] = s[3] = -INFINITY, ub = make_uint2(0, 0);
      }
      const bool above = s[0] > top[0] || s[2] > top[0] || s[1] > top[1] || s[3] > top[1];
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(m[e], fmaxf(s[e], s[e + 2]));
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float alpha = ex2(m[e] - mx);
          m[e] = mx;
          top[e] = mx + kKv4Slack;
          l[e] *= alpha;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i][e] *= alpha, o[i][e + 2] *= alpha;
        }
      }
      float pr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pr[i] = ex2(s[i] - m[i & 1]);
      l[0] += pr[0] + pr[2];
      l[1] += pr[1] + pr[3];
      const float ga[4] = {bf16lo_to_f32(ua.x), bf16hi_to_f32(ua.x), bf16lo_to_f32(ua.y), bf16hi_to_f32(ua.y)};
      const float gb[4] = {bf16lo_to_f32(ub.x), bf16hi_to_f32(ub.x), bf16lo_to_f32(ub.y), bf16hi_to_f32(ub.y)};
      const uint8_t* vt = buf + kKv4CodeBytes + (t / 2 + tig) * 128 + ((gid ^ (2 * tig)) * 16);
      const uint4 va = *reinterpret_cast<const uint4*>(vt), vb = *reinterpret_cast<const uint4*>(vt + 4 * 128);
      const uint32_t xa[4] = {va.x, va.y, va.z, va.w}, xb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x0 = pr[0] * ga[j], x1 = pr[1] * ga[j], x2 = pr[2] * gb[j], x3 = pr[3] * gb[j];
        const uint32_t p0 = pack_bf16x2(x0, x1), p1 = pack_bf16x2(x2, x3);
        const uint32_t b0 = movmatrix_trans(p0), b1 = movmatrix_trans(p1);
        const uint32_t v0 = nibbles_code<0>(xa[j], magic), v1 = nibbles_code<1>(xa[j], magic);
        const uint32_t v2 = nibbles_code<0>(xb[j], magic), v3 = nibbles_code<1>(xb[j], magic);
        const uint32_t v4 = nibbles_code<2>(xa[j], magic), v5 = nibbles_code<3>(xa[j], magic);
        const uint32_t v6 = nibbles_code<2>(xb[j], magic), v7 = nibbles_code<3>(xb[j], magic);
        mma_bf16_acc(o[2 * j], v0, v1, v2, v3, b0, b1);
        mma_bf16_acc(o[2 * j + 1], v4, v5, v6, v7, b0, b1);
        const uint32_t r0 = movmatrix_trans(pack_bf16x2(x0 - bf16lo_to_f32(p0), x1 - bf16hi_to_f32(p0)));
        const uint32_t r1 = movmatrix_trans(pack_bf16x2(x2 - bf16lo_to_f32(p1), x3 - bf16hi_to_f32(p1)));
        mma_bf16_acc(o[2 * j], v0, v1, v2, v3, r0, r1);
        mma_bf16_acc(o[2 * j + 1], v4, v5, v6, v7, r0, r1);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
    bool fed = true;
    if (tid == 0 && left > kKv4Stages) {
      fed = mbar_wait(&empty[st], round, kErrTimeoutEmpty);
      if (fed) feed_unit();
    }
    if (!__all_sync(0xffffffffu, fed)) return drain();
    if (++st == kKv4Stages) st = 0, round ^= 1;

    if (mt.last) {  // join the warps
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
      const int b = mt.job / p.Hkv, h0 = (mt.job - b * p.Hkv) * G;
      float* slot = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (mt.last == 3)) * kKv4SlotFloats;
      for (int g0 = 0; g0 < G; g0 += 4, ++merges) {  // four heads at a time
        if (merges > 0 && !mbar_wait(&red_free, (merges - 1) & 1, kErrTimeoutEmpty)) return drain();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int head = 2 * tig + e;
          if (head >= g0 && head < min(G, g0 + 4)) {
            float* dst = red + (warp * 4 + head - g0) * kKv4RedStride + gid * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(dst + 32 * j) =
                  make_float4(o[2 * j][e], o[2 * j][e + 2], o[2 * j + 1][e], o[2 * j + 1][e + 2]);
            if (gid == 0) red_ml[warp][head][0] = m[e], red_ml[warp][head][1] = l[e];
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_full);
        if (!mbar_wait(&red_full, merges & 1, kErrTimeoutFull)) return drain();
        const int d = tid % kKv4D;
        for (int head = g0 + tid / kKv4D; head < min(G, g0 + 4); head += kKv4Threads / kKv4D) {
          float M = kKv4NoMax, S = 0.0f, acc = 0.0f;
#pragma unroll
          for (int w = 0; w < kKv4Warps; ++w) M = fmaxf(M, red_ml[w][head][0]);
#pragma unroll
          for (int w = 0; w < kKv4Warps; ++w) {
            const float f = ex2(red_ml[w][head][0] - M);
            S = fmaf(f, red_ml[w][head][1], S);
            acc = fmaf(f, red[(w * 4 + head - g0) * kKv4RedStride + d], acc);
          }
          if (mt.last == 1) {
            p.out[(static_cast<int64_t>(b) * p.Hq + h0 + head) * kKv4D + d] =
                __bfloat16_as_ushort(__float2bfloat16_rn(S == 0.0f ? 0.0f : acc / S));
          } else {
            slot[head * kKv4D + d] = acc;
            if (d == 0) *reinterpret_cast<float2*>(slot + kKv4MaxGroup * kKv4D + 2 * head) = make_float2(M, S);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_free);
      }
    }
  }
}
static_assert(kKv4Threads % kKv4D == 0, "the join takes a channel a thread");

// Joins the partials of the jobs that several CTAs hold, and writes the zeros of
// empty sequences.  One CTA per (sequence, query head), a thread per channel, or
// four that take every fourth part where a job is spread over many CTAs (a single
// 32k sequence: 74 parts).  Latency bound, so two rounds of loads: the cuts; the
// maxima and sums, one part a thread, with the first eight outputs of each thread.
constexpr int kKv4MergeGroups = 4;
__global__ void __launch_bounds__(kKv4MergeGroups * kKv4D) kv4_merge_kernel(const Kv4AttnArgs p, int grid) {
  __shared__ float weight[kKv4MaxCtas], most[kKv4MergeGroups * 4], sums[kKv4MergeGroups * 4];
  __shared__ float part_acc[kKv4MergeGroups][kKv4D];
  const int b = blockIdx.x / p.Hq, hq = blockIdx.x - b * p.Hq, G = p.Hq / p.Hkv, h = hq / G, g = hq - h * G;
  const int tid = threadIdx.x, d = tid % kKv4D, group = tid / kKv4D, groups = blockDim.x / kKv4D;
  const int lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  grid_dependency_wait();
  const int64_t first = p.starts[b], n = p.starts[b + 1] - first, total = p.starts[p.B] * p.Hkv;
  uint16_t* out = p.out + static_cast<int64_t>(blockIdx.x) * kKv4D + d;
  if (n == 0) {
    if (group == 0) *out = 0;
    return;
  }
  const int ctas = static_cast<int>(min(total, static_cast<int64_t>(grid)));
  const int64_t a = first * p.Hkv + h * n, e = a + n;
  // the CTA of a unit u is the largest i whose cut is at or before it
  const int c0 = static_cast<int>(((a + 1) * ctas + total - 1) / total) - 1;
  const int c1 = static_cast<int>((e * ctas + total - 1) / total) - 1;
  if (c0 == c1) return;
  // c0 holds its part in slot 0 when the job is the first of its units, the others always do
  const int parts = c1 - c0 + 1;
  const float* at = p.partials + (2 * static_cast<int64_t>(c0)) * kKv4SlotFloats;
  const int64_t skew = kv4_cut(total, c0, ctas) < a ? kKv4SlotFloats : 0;  // of part 0
  const auto part = [&](int i) { return at + i * (2 * kKv4SlotFloats) + (i == 0 ? skew : 0); };
  float v[8];
  const auto load = [&](int i0) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int i = i0 + x * groups;
      v[x] = i < parts ? part(i)[g * kKv4D + d] : 0.0f;
    }
  };
  load(group);
  const int kMl = kKv4MaxGroup * kKv4D + 2 * g;
  float mx = kKv4NoMax;
  for (int i = tid; i < parts; i += blockDim.x) mx = fmaxf(mx, part(i)[kMl]);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  if (lane == 0) most[warp] = mx;
  __syncthreads();
  for (int w = 0; w < warps; ++w) mx = fmaxf(mx, most[w]);
  float fs = 0.0f;
  for (int i = tid; i < parts; i += blockDim.x) {
    const float2 ml = *reinterpret_cast<const float2*>(part(i) + kMl);
    const float f = ex2(ml.x - mx);
    weight[i] = f;
    fs = fmaf(f, ml.y, fs);
  }
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) fs += __shfl_xor_sync(0xffffffffu, fs, x);
  if (lane == 0) sums[warp] = fs;
  __syncthreads();
  float S = 0.0f, acc = 0.0f;
  for (int w = 0; w < warps; ++w) S += sums[w];
  for (int i0 = group; i0 < parts; i0 += 8 * groups) {
    if (i0 != group) load(i0);
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (i0 + x * groups < parts) acc = fmaf(weight[i0 + x * groups], v[x], acc);
  }
  if (groups > 1) {
    part_acc[group][d] = acc;
    __syncthreads();
    if (group != 0) return;
    for (int i = 1; i < groups; ++i) acc += part_acc[i][d];
  }
  *out = __bfloat16_as_ushort(__float2bfloat16_rn(S == 0.0f ? 0.0f : acc / S));
}

static int64_t kv4_starts_bytes(int64_t batch) { return (batch + 1) * 8 + 15 & ~int64_t(15); }
static int64_t kv4_max_ctas(int64_t batch, int64_t num_heads, int64_t max_pages) {
  return std::min<int64_t>(kKv4MaxCtas, batch * num_heads * max_pages * (kKv4Page / kKv4Unit));
}
int64_t paged_attention_kv4_workspace_bytes(int64_t batch, int64_t num_heads, int64_t max_pages) {
  return kv4_starts_bytes(batch) + kv4_max_ctas(batch, num_heads, max_pages) * 2 * kKv4SlotFloats * 4;
}

int launch_paged_decode_attention_kv4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                      const void* v_scales, const int* block_tables, const int* context_lens,
                                      void* out, void* workspace, int64_t batch, int64_t num_heads,
                                      int64_t num_kv_heads, int64_t num_pages, int64_t max_pages, float scale,
                                      cudaStream_t stream) {
  static int done[64] = {};
  const auto kernel = paged_decode_attention_kv4_kernel;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kernel), kKv4Smem, done);
  if (rc != NV4_OK) return rc;
  Kv4AttnArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k_codes = static_cast<const uint8_t*>(k_codes);
  a.k_scales = static_cast<const uint16_t*>(k_scales);
  a.v_codes = static_cast<const uint8_t*>(v_codes);
  a.v_scales = static_cast<const uint16_t*>(v_scales);
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.out = static_cast<uint16_t*>(out);
  a.starts = static_cast<int64_t*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kv4_starts_bytes(batch));
  a.num_pages = num_pages;
  a.B = static_cast<int>(batch);
  a.Hq = static_cast<int>(num_heads);
  a.Hkv = static_cast<int>(num_kv_heads);
  a.max_pages = static_cast<int>(max_pages);
  a.scale_log2 = scale * 1.4426950408889634f;
  // no more CTAs than there can be units
  const int ctas = static_cast<int>(std::min<int64_t>(
      kv4_max_ctas(batch, num_kv_heads, max_pages), kKv4CtasPerSm * static_cast<int64_t>(device_sm_count())));
  rc = launch_kernel(kernel, dim3(ctas), dim3(kKv4Threads), kKv4Smem, stream, false, a);
  if (rc != NV4_OK) return rc;
  // more than eight parts a job at the most: four threads a channel
  const int groups = ctas > 8 * batch * num_kv_heads ? kKv4MergeGroups : 1;
  return launch_kernel(kv4_merge_kernel, dim3(static_cast<unsigned>(batch * num_heads)), dim3(groups * kKv4D), 0, stream,
                       true, a, ctas);
}

}  // namespace nv4
