// The quantised paged KV cache: writing, reading, page selection, and the C entry points (include/piper_cache.h).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache_kernels.h"
#include "host.h"
#include "piper_cache.h"

namespace piper {
namespace {

// ---- write and read -------------------------------------------------------------------------------------------------
//
// Both are bound by the bytes they move.  A workgroup has a page of one K/V head, each wave groups of eight of its tokens:
// lane 8 r + c has an eighth of token r's features, in 32 (D = 128) or 16 consecutive bytes of 16-bit values.  Key
// codes lie as the lanes have them; value codes change lanes, so that each has all eight tokens of two features or one.
// Four sequences' 8192 tokens of 8 heads of 128: the write 52 us for 201 MB, 3.9 TB/s, the read 33.  (A token a lane with
// value codes stored byte by byte: 198 us for the two.)  A pass of the two, 94 us, took 102 with eight waves a workgroup of
// the write, 98 with the next tokens' loads ahead, 101 with those and two waves, 107 with 64 registers for eight waves a SIMD (13
// spilled).  One token for each of 64 sequences: 8.4 us, a chain of loads.

constexpr int kMoveWaves = 4;

template <int kDim>
struct Eighth {  // of a token's row
  static constexpr int kValues = kDim / 8, kLoads = kDim / 64, kWords = kDim / 32;  // 16-byte loads; words of four codes
};

// Swaps the values of two registers between lanes 32 (16) apart: the lower lanes end with both lanes' `a`, the upper ones
// with both lanes' `b`, the lower lane's first.
__device__ __forceinline__ void exchange32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

__device__ __forceinline__ void exchange16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

__device__ __forceinline__ uint32_t lane_xor8(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xf, 0xf, false));  // row_ror:8
}

// Bytes of two words by selector (0-3: of b, 4-7: of a).
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t selector) { return __builtin_amdgcn_perm(a, b, selector); }

// From lane 8 r + c's codes of token r, features kValues c .. + kValues - 1, those of tokens 0..7 of features
// (kValues / 8) (8 c + r) .. : halves of the words change lanes with r's top bit, halves of the rest with the next, and the
// last step, lanes 8 apart, interleaves the even tokens' bytes with the odd ones'.
template <int kDim>
__device__ __forceinline__ void tokens_together(const uint32_t (&codes)[kDim / 32], uint32_t (&out)[kDim / 32], int r) {
  uint32_t mine[kDim / 64], other[kDim / 64];  // tokens t, t + 2 | t + 4, t + 6 (t = r % 2) of this lane's feature(s), and of its partner's
  if constexpr (kDim == 128) {
    uint32_t p0 = codes[0], p1 = codes[2], q0 = codes[1], q1 = codes[3];
    exchange32(p0, p1);
    exchange32(q0, q1);
    exchange16(p0, q0);  // tokens t, t + 2
    exchange16(p1, q1);  // tokens t + 4, t + 6
    const uint32_t low0 = bytes_of(q0, p0, 0x05040100), high0 = bytes_of(q0, p0, 0x07060302);
    const uint32_t low1 = bytes_of(q1, p1, 0x05040100), high1 = bytes_of(q1, p1, 0x07060302);
    mine[0] = r & 1 ? high0 : low0;
    mine[1] = r & 1 ? high1 : low1;
    other[0] = lane_xor8(r & 1 ? low0 : high0);
    other[1] = lane_xor8(r & 1 ? low1 : high1);
    const uint32_t even0 = r & 1 ? other[0] : mine[0], odd0 = r & 1 ? mine[0] : other[0];
    const uint32_t even1 = r & 1 ? other[1] : mine[1], odd1 = r & 1 ? mine[1] : other[1];
    out[0] = bytes_of(odd0, even0, 0x06020400);
    out[1] = bytes_of(odd1, even1, 0x06020400);
    out[2] = bytes_of(odd0, even0, 0x07030501);
    out[3] = bytes_of(odd1, even1, 0x07030501);
  } else {
    uint32_t p0 = codes[0], p1 = codes[1];
    exchange32(p0, p1);  // tokens t, t + 4 (t = r % 4)
    uint32_t low = bytes_of(p1, p0, 0x05040100), high = bytes_of(p1, p0, 0x07060302);
    exchange16(low, high);  // tokens t, t + 4 | t + 2, t + 6 (t = r % 2) of two features
    const uint32_t first = bytes_of(high, low, 0x06020400), second = bytes_of(high, low, 0x07030501);  // tokens t, t + 2, t + 4, t + 6
    mine[0] = r & 1 ? second : first;
    other[0] = lane_xor8(r & 1 ? first : second);
    const uint32_t even = r & 1 ? other[0] : mine[0], odd = r & 1 ? mine[0] : other[0];
    out[0] = bytes_of(odd, even, 0x05010400);
    out[1] = bytes_of(odd, even, 0x07030602);
  }
}

// Max over the eight lanes of a token.
__device__ __forceinline__ uint32_t token_max(uint32_t v) {
  const auto max_with = [&](auto ctrl) {
    const uint32_t x = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, false));
    v = v > x ? v : x;
  };
  max_with(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  max_with(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  max_with(std::integral_constant<int, 0x141>{});  // row_half_mirror
  return v;
}

typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));

// A token's codes from its 16-bit values, and its scale.  Largest magnitude: the values' bits without the sign are in
// the order of whole numbers, infinities and NaN above all.
template <bool kBf16, bool kFp8, int kDim>
__device__ __forceinline__ float encode_row(const uint4 (&raw)[kDim / 64], uint32_t (&codes)[kDim / 32]) {
  ushort2_t most = {0, 0};
#pragma unroll
  for (int k = 0; k < kDim / 64; ++k) {
    const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(ushort2_t, w[i] & 0x7fff7fffu));
  }
  const uint32_t bits = token_max(most.x > most.y ? most.x : most.y);
  const RowCode code = row_code<kFp8>(widen<kBf16>(static_cast<uint16_t>(bits)), bits < (kBf16 ? 0x7f80u : 0x7c00u));
#pragma unroll
  for (int k = 0; k < kDim / 64; ++k) {
    float x[8];
    widen8<kBf16>(code.inv == 0.0f ? uint4{0, 0, 0, 0} : raw[k], x);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if constexpr (kFp8) {
        int packed = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w] * code.inv, x[4 * w + 1] * code.inv, 0, false);
        codes[2 * k + w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2] * code.inv, x[4 * w + 3] * code.inv, packed, true));
      } else {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma clang fp contract(off)  // see code_of_value
          c[i] = __float_as_uint(x[4 * w + i] * code.inv + kAccBiasValue);
        }
        codes[2 * k + w] = bytes_of(bytes_of(c[3], c[2], 0x0c0c0400), bytes_of(c[1], c[0], 0x0c0c0400), 0x05040100);
      }
    }
  }
  return code.scale;
}

template <bool kFp8>
__device__ __forceinline__ void decode4(uint32_t codes, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFp8) {
      switch (i) {
        case 0: x[i] = __builtin_amdgcn_cvt_f32_fp8(codes, 0); break;
        case 1: x[i] = __builtin_amdgcn_cvt_f32_fp8(codes, 1); break;
        case 2: x[i] = __builtin_amdgcn_cvt_f32_fp8(codes, 2); break;
        default: x[i] = __builtin_amdgcn_cvt_f32_fp8(codes, 3); break;
      }
    } else {
      x[i] = static_cast<float>(static_cast<int8_t>(codes >> (8 * i)));
    }
  }
}

// Codes of the rows of a page of one K/V head; of a page that they fill also its bounds.
template <bool kBf16, bool kFp8, int kDim>
__global__ __launch_bounds__(kWave* kMoveWaves) void cache_write_kernel(CacheMove a) {
  using E = Eighth<kDim>;
  __shared__ float ends[kMoveWaves][2][kDim];
  __shared__ float tops[2];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r = lane / 8, c = lane % 8;
  const int64_t touched = pages_touched(a.rows.tokens);
  const int64_t unit = blockIdx.x / touched;
  const int64_t b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int64_t logical = floor_page(a.rows.start(b)) + blockIdx.x % touched;
  const PageRows in = rows_in_page(a.rows, b, logical);
  const int64_t page = a.rows.page(b, logical);
  if (in.n == 0 || page < 0) return;
  const int64_t record = page * a.cache.kv_heads + h;
  uint8_t* const keys = a.cache.key + record * (kPage * kDim);
  uint8_t* const values = a.cache.value + record * (kPage * kDim);
  const bool fills = in.slot + in.n == kPage;
  const int begin = fills ? 0 : in.slot / 8, end = (in.slot + in.n + 7) / 8;
  const uint16_t* const key_rows = static_cast<const uint16_t*>(a.key.data) + b * a.key.stride_batch + h * a.key.stride_head + E::kValues * c;
  const uint16_t* const value_rows = static_cast<const uint16_t*>(a.value.data) + b * a.value.stride_batch + h * a.value.stride_head + E::kValues * c;
  float upper[E::kValues], lower[E::kValues];
#pragma unroll
  for (int i = 0; i < E::kValues; ++i) upper[i] = -__builtin_inff(), lower[i] = __builtin_inff();

  for (int eight = begin + wave; eight < end; eight += kMoveWaves) {
    const int slot = 8 * eight + r;
    const bool mine = slot >= in.slot && slot < in.slot + in.n;  // a row of the call
    const int64_t row = in.first + (mine ? slot - in.slot : 0);
    uint4 key[E::kLoads], value[E::kLoads];
#pragma unroll
    for (int k = 0; k < E::kLoads; ++k) {
      key[k] = *reinterpret_cast<const uint4*>(key_rows + row * a.key.stride_seq + 8 * k);
      value[k] = *reinterpret_cast<const uint4*>(value_rows + row * a.value.stride_seq + 8 * k);
    }
    uint32_t codes[E::kWords], tokens[E::kWords];
    float scale = encode_row<kBf16, kFp8, kDim>(value, codes);
    tokens_together<kDim>(codes, tokens, r);
    uint8_t* const to = values + eight * (8 * kDim) + (8 * c + r) * kDim / 8;
    if (8 * eight >= in.slot && 8 * eight + 8 <= in.slot + in.n) {
      if constexpr (kDim == 128)
        *reinterpret_cast<uint4*>(to) = uint4{tokens[0], tokens[1], tokens[2], tokens[3]};
      else
        *reinterpret_cast<uint2*>(to) = uint2{tokens[0], tokens[1]};
    } else {  // the other slots' bytes stay
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        if (8 * eight + t < in.slot || 8 * eight + t >= in.slot + in.n) continue;
#pragma unroll
        for (int f = 0; f < kDim / 64; ++f) to[8 * f + t] = static_cast<uint8_t>(tokens[2 * f + t / 4] >> (8 * (t % 4)));
      }
    }
    if (mine && c == 0) a.cache.value_scale[record * kPage + slot] = scale;
    scale = encode_row<kBf16, kFp8, kDim>(key, codes);
    uint8_t* const key_to = keys + slot * kDim + E::kValues * c;
    if (mine) {
      if constexpr (kDim == 128)
        *reinterpret_cast<uint4*>(key_to) = uint4{codes[0], codes[1], codes[2], codes[3]};
      else
        *reinterpret_cast<uint2*>(key_to) = uint2{codes[0], codes[1]};
      if (c == 0) a.cache.key_scale[record * kPage + slot] = scale;
    } else if (fills) {  // a full page's earlier keys, for its bounds
      scale = a.cache.key_scale[record * kPage + slot];
#pragma unroll
      for (int w = 0; w < E::kWords; ++w) codes[w] = reinterpret_cast<const uint32_t*>(key_to)[w];
    }
    if (fills) {
#pragma unroll
      for (int w = 0; w < E::kWords; ++w) {
        float x[4];
        decode4<kFp8>(codes[w], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float k = x[i] * scale;  // NaN is left out
          upper[4 * w + i] = fmaxf(upper[4 * w + i], k);
          lower[4 * w + i] = fminf(lower[4 * w + i], k);
        }
      }
    }
  }
  if (!fills) return;
#pragma unroll
  for (int i = 0; i < E::kValues; ++i) {  // over a wave's tokens: lanes 8, 16 and 32 apart
    upper[i] = fmaxf(upper[i], __uint_as_float(lane_xor8(__float_as_uint(upper[i]))));
    lower[i] = fminf(lower[i], __uint_as_float(lane_xor8(__float_as_uint(lower[i]))));
    uint32_t u = __float_as_uint(upper[i]), v = __float_as_uint(upper[i]);
    exchange16(u, v);
    upper[i] = fmaxf(__uint_as_float(u), __uint_as_float(v));
    u = v = __float_as_uint(upper[i]);
    exchange32(u, v);
    upper[i] = fmaxf(__uint_as_float(u), __uint_as_float(v));
    u = v = __float_as_uint(lower[i]);
    exchange16(u, v);
    lower[i] = fminf(__uint_as_float(u), __uint_as_float(v));
    u = v = __float_as_uint(lower[i]);
    exchange32(u, v);
    lower[i] = fminf(__uint_as_float(u), __uint_as_float(v));
    if (r == 0) {
      ends[wave][0][E::kValues * c + i] = upper[i];
      ends[wave][1][E::kValues * c + i] = lower[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < kDim) {
    float up = ends[0][0][threadIdx.x], low = ends[0][1][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kMoveWaves; ++w) up = fmaxf(up, ends[w][0][threadIdx.x]), low = fminf(low, ends[w][1][threadIdx.x]);
    if (up < low) up = low = 0.0f;  // every key of the page is NaN
    ends[0][0][threadIdx.x] = up;
    ends[0][1][threadIdx.x] = low;
    const float top = wave_max(fmaxf(fabsf(up), fabsf(low)));
    if (lane == 0) tops[wave] = top;
  }
  __syncthreads();
  if (threadIdx.x < kDim) {
    const RowCode code = row_code<false>(kDim == 128 ? fmaxf(tops[0], tops[1]) : tops[0], true);
    int8_t* const to = a.cache.bounds + record * 2 * kDim + threadIdx.x;
    to[0] = static_cast<int8_t>(code_of_value<false>(ends[0][0][threadIdx.x], code.inv));
    to[kDim] = static_cast<int8_t>(code_of_value<false>(ends[0][1][threadIdx.x], code.inv));
    if (threadIdx.x == 0) a.cache.bound_scale[record] = code.scale;
  }
}

// Two values' products in FP32, then the output's rounding. For FP16 the compiler would make one instruction of the
// two (v_fma_mixlo_f16, one rounding, whatever the contraction mode), and a few values would differ by an ulp from
// what the cache is defined to hold: the products are pinned in registers between.
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow_product2(float x, float y, float scale) {
  float a = x * scale, b = y * scale;
  if constexpr (!kBf16) asm("" : "+v"(a), "+v"(b));
  return narrow2<kBf16>(a, b);
}

template <bool kBf16, bool kFp8>
__device__ __forceinline__ uint2 decode_row4(uint32_t codes, float scale) {
  float x[4];
  decode4<kFp8>(codes, x);
  return uint2{narrow_product2<kBf16>(x[0], x[1], scale), narrow_product2<kBf16>(x[2], x[3], scale)};
}

// Values of the rows of a page of one K/V head, and zeros for those of them that are padding or have no page.
template <bool kBf16, bool kFp8, int kDim>
__global__ __launch_bounds__(kWave* kMoveWaves) void cache_read_kernel(CacheMove a) {
  using E = Eighth<kDim>;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, r = lane / 8, c = lane % 8;
  const int64_t touched = pages_touched(a.rows.tokens);
  const int64_t unit = blockIdx.x / touched;
  const int64_t b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int64_t start = a.rows.start(b), logical = floor_page(start) + blockIdx.x % touched, base = logical * kPage;
  const int count = a.rows.count(b);
  const int64_t page = a.rows.page(b, logical);
  const int64_t record = (page >= 0 ? page : 0) * a.cache.kv_heads + h;
  uint16_t* const key_out = static_cast<uint16_t*>(const_cast<void*>(a.key.data)) + unit * a.rows.tokens * kDim;
  uint16_t* const value_out = static_cast<uint16_t*>(const_cast<void*>(a.value.data)) + unit * a.rows.tokens * kDim;
  const uint8_t* const keys = a.cache.key + record * (kPage * kDim);
  const uint8_t* const values = a.cache.value + record * (kPage * kDim);
#pragma unroll
  for (int k = 0; k < 8 / kMoveWaves; ++k) {
    const int eight = wave + k * kMoveWaves;
    // rows base - start + slot of the call, of which [0, tokens) exist
    const int64_t first = base - start + 8 * eight;
    if (first + 8 <= 0 || first >= a.rows.tokens) continue;
    {
      const int slot = 8 * eight + r;
      const int64_t row = first + r;
      const float held = a.cache.key_scale[record * kPage + slot];
      uint32_t codes[E::kWords];
#pragma unroll
      for (int w = 0; w < E::kWords; ++w) codes[w] = reinterpret_cast<const uint32_t*>(keys + slot * kDim + E::kValues * c)[w];
      const bool real = page >= 0 && row < count;
      if (row >= 0 && row < a.rows.tokens) {
#pragma unroll
        for (int w = 0; w < E::kWords; w += 2) {
          const uint2 x = decode_row4<kBf16, kFp8>(codes[w], held), y = decode_row4<kBf16, kFp8>(codes[w + 1], held);
          *reinterpret_cast<uint4*>(key_out + row * kDim + E::kValues * c + 4 * w) = real ? uint4{x.x, x.y, y.x, y.y} : uint4{0, 0, 0, 0};
        }
      }
    }
    // values: a lane's eight tokens of features 2 lane and 2 lane + 1, or of feature lane
    uint32_t codes[E::kWords];
#pragma unroll
    for (int w = 0; w < E::kWords; ++w) codes[w] = reinterpret_cast<const uint32_t*>(values + eight * (8 * kDim) + lane * (kDim / 8))[w];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float4 held = *reinterpret_cast<const float4*>(a.cache.value_scale + record * kPage + 8 * eight + 4 * half);
      const float scale[4] = {held.x, held.y, held.z, held.w};
      float x[4], y[4] = {};
      decode4<kFp8>(codes[half], x);
      if constexpr (kDim == 128) decode4<kFp8>(codes[2 + half], y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = first + 4 * half + i;
        if (row < 0 || row >= a.rows.tokens) continue;
        const uint32_t packed = page >= 0 && row < count ? narrow_product2<kBf16>(x[i], y[i], scale[i]) : 0u;
        if constexpr (kDim == 128)
          reinterpret_cast<uint32_t*>(value_out + row * kDim)[lane] = packed;
        else
          value_out[row * kDim + lane] = static_cast<uint16_t>(packed);
      }
    }
  }
}

// ---- selection ------------------------------------------------------------------------------------------------------
//
// A score's sum over the features of max(c, 0) upper + min(c, 0) lower is one integer product of a page's bounds, which
// lie in memory as the 2 D bytes that a 16x16x64 instruction takes row by row, with [q+, q-].  Its columns are a K/V
// head's query heads, token by token; the maximum over a token's columns is one over lanes.  The scores go to LDS and a
// wave (or for one token all waves) picks the token's pages from registers: the last one's score is found bit by bit,
// counting with ballots, and the pages come out in their order.  Reading the bounds is what a single token's call has to
// do; in a chunk the picking, about 20 counts of n / 64 ballots a row, costs as much.  64 of up to 1024 pages for 128 rows: 11.8 us
// for the scores (21 MB), 13 for the pages; three bits of a score for each barrier (28 us before, one bit each).  32 of
// 264 pages for 2000 rows: 20 us.

typedef int int4_t __attribute__((ext_vector_type(4)));

constexpr int kSelectWaves = 8;
constexpr int kRowScores = 16384;  // scores in LDS: 64 KiB, two workgroups a CU; also what a workgroup's registers hold
constexpr int kWaveScores = 1024;  // what one wave's registers hold
constexpr int kShortWaves = 4, kShortPages = 64;  // of a wave alone: four tiles, which it scores at once

// Scores in the order of whole numbers: the larger the score, the larger the number (-0 is 0, NaN -infinity); all of
// them above 0, which stands for no score.
__device__ __forceinline__ uint32_t score_order(float score) {
  const uint32_t u = __float_as_uint(fmaxf(score, -__builtin_inff()) + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Where a row of the call stands: its own page, -1 for a row that is none or stands where the table does not reach.
__device__ __forceinline__ int own_page(const CacheSelect& a, int64_t b, int64_t i) {
  if (i >= a.rows.count(b)) return -1;
  const int64_t end = a.rows.end(b, i);
  return end > 0 && end == a.rows.start(b) + i + 1 ? static_cast<int>((end - 1) / kPage) : -1;
}

// Scores of pages [from, to) for `tokens` rows from `first` on, a wave's tiles of 16 pages being `stride` apart.
// store(token, page, score).
template <bool kBf16, int kDim, typename Store>
__device__ __forceinline__ void score_pages(const CacheSelect& a, int64_t b, int64_t h, int first, int tokens, int columns, int from, int to,
                                            int stride, Store store) {
  constexpr int kParts = kDim / 64, kBatch = 4;
  const int lane = threadIdx.x % kWave, n = lane % 16, g = lane / 16;
  const int group = a.heads / a.cache.kv_heads;
  for (int tile = from; tile < to; tile += kBatch * stride) {
    int4_t bounds[kBatch][2 * kParts];
    float scale[kBatch];
    bool there[kBatch];
#pragma unroll
    for (int t = 0; t < kBatch; ++t) {
      const int page = tile + t * stride + n;
      const int64_t p = page < to ? a.rows.page(b, page) : -1;
      there[t] = p >= 0;
      const int64_t record = (there[t] ? p : 0) * a.cache.kv_heads + h;
      const int8_t* const at = a.cache.bounds + record * 2 * kDim + 16 * g;
#pragma unroll
      for (int k = 0; k < 2 * kParts; ++k) bounds[t][k] = *reinterpret_cast<const int4_t*>(at + 64 * k);
      scale[t] = a.cache.bound_scale[record];
    }
    float best[kBatch][4];
    for (int round = 0; round * columns < group; ++round) {
      // column n: a head's row in the two halves' codes
      const int token = first + n / columns, head = round * columns + n % columns;
      const bool real = n / columns < tokens && head < group;
      const uint16_t* q = static_cast<const uint16_t*>(a.query.data) + b * a.query.stride_batch;
      if (real) q += (h * group + head) * a.query.stride_head + token * a.query.stride_seq;
      float x[kParts][16], top = 0.0f;
      bool finite = true;
#pragma unroll
      for (int k = 0; k < kParts; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float half[8];
          widen8<kBf16>(*reinterpret_cast<const uint4*>(q + 64 * k + 16 * g + 8 * e), half);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[k][8 * e + i] = half[i];
            top = fmaxf(top, fabsf(half[i]));
            finite = finite && is_finite(half[i]);
          }
        }
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const uint64_t good = __ballot(finite);
      const RowCode code = row_code<false>(top, (good >> n & 0x0001000100010001ull) == 0x0001000100010001ull);
      int4_t codes[2 * kParts];
#pragma unroll
      for (int k = 0; k < kParts; ++k)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t plus = 0, minus = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t c = code_of_value<false>(x[k][4 * w + i], code.inv);
            plus |= (c < 128 ? c : 0) << (8 * i);
            minus |= (c < 128 ? 0 : c) << (8 * i);
          }
          codes[k][w] = static_cast<int>(plus);
          codes[kParts + k][w] = static_cast<int>(minus);
        }
#pragma unroll
      for (int t = 0; t < kBatch; ++t) {
        int4_t dot = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 2 * kParts; ++k) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(bounds[t][k], codes[k], dot, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float s = real ? __fmul_rn(static_cast<float>(dot[i]), code.scale) : -__builtin_inff();
          best[t][i] = round > 0 ? fmaxf(best[t][i], s) : s;
        }
      }
    }
    // a token's columns, then the pages' scales: row 4 g + i of a tile is its page
#pragma unroll
    for (int t = 0; t < kBatch; ++t) {
      const uint64_t named = __ballot(there[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s = best[t][i];
        for (int m = columns / 2; m >= 1; m /= 2) s = fmaxf(s, __shfl_xor(s, m, kWave));
        s = __fmul_rn(s, __shfl(scale[t], 4 * g + i, kWave));
        const int row = 4 * g + i, page = tile + t * stride + row;
        if (n % columns == 0 && n / columns < tokens && page < to) store(n / columns, page, named >> row & 1 ? s : -__builtin_inff());
      }
    }
  }
}

// Counts of all waves (kAll; else of this one).
constexpr int kCountWords = 2 * kSelectWaves;  // of LDS: two counts in turn, one barrier each

template <bool kAll>
__device__ __forceinline__ uint4 count_all(uint4 mine, uint4* shared, int& turn) {
  if constexpr (!kAll) return mine;
  uint4* const of = shared + (turn++ & 1) * kSelectWaves;
  if (threadIdx.x % kWave == 0) of[threadIdx.x / kWave] = mine;
  __syncthreads();
  uint4 sum = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    const uint4 x = of[w];
    sum = uint4{sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w};
  }
  return sum;
}

template <bool kAll>
__device__ __forceinline__ int count_all(int mine, uint4* shared, int& turn) {
  return static_cast<int>(count_all<kAll>(uint4{static_cast<uint32_t>(mine), 0, 0, 0}, shared, turn).x);
}

// The largest number that at least `wanted` of `all` orders reach, digit by digit from the top, or any that just `wanted`
// do; `reach`: how many.  count(number) is a wave's count of orders that reach a number.  A digit of kBits costs
// 2^kBits - 1 counts and, over all waves, one barrier; with kBits > 1
// two counts share a word, and all stay below 2^16.
template <bool kAll, int kBits, typename Count>
__device__ __forceinline__ uint32_t least_order(int wanted, int all, int& reach, uint4* shared, int& turn, Count count) {
  static_assert(kBits >= 1 && kBits <= 3, "seven counts in four words");
  uint32_t least = 0;
  reach = all;
  for (int shift = 32; shift > 0 && reach != wanted;) {
    const int bits = shift % kBits == 0 ? kBits : shift % kBits;  // the first digit may be short
    shift -= bits;
    uint32_t mine[8] = {};
#pragma unroll
    for (int d = 1; d < 1 << kBits; ++d)
      if (d < 1 << bits) mine[d] = count(least + (static_cast<uint32_t>(d) << shift));
    if constexpr (kBits == 1) {
      const int sum = count_all<kAll>(static_cast<int>(mine[1]), shared, turn);
      if (sum >= wanted) {
        least += 1u << shift;
        reach = sum;
      }
      continue;
    }
    const uint4 sum = count_all<kAll>(uint4{mine[1] | mine[2] << 16, mine[3] | mine[4] << 16, mine[5] | mine[6] << 16, mine[7]}, shared, turn);
    const uint32_t of[8] = {0, sum.x & 0xffffu, sum.x >> 16, sum.y & 0xffffu, sum.y >> 16, sum.z & 0xffffu, sum.z >> 16, sum.w};
    int digit = 0;
#pragma unroll
    for (int d = 1; d < 1 << kBits; ++d)
      if (d < 1 << bits && static_cast<int>(of[d]) >= wanted) {
        digit = d;
        reach = of[d];
      }
    least += static_cast<uint32_t>(digit) << shift;
  }
  return least;
}

// Writes a row's pages: of its `earlier` scores the budget - 1 largest, ties to the lower page, and `own`.  By one wave, or by
// all of the workgroup's, each with kHeld runs of 64 scores.
template <bool kAll, int kHeld>
__device__ __forceinline__ void pick_pages(const float* scores, int own, int budget, int32_t* out, uint4* shared, int& turn) {
  const int lane = threadIdx.x % kWave, wave = kAll ? threadIdx.x / kWave : 0;
  const int earlier = own > 0 ? own : 0, wanted = earlier < budget - 1 ? earlier : budget - 1;
  const int base = wave * kHeld * kWave;
  if (wanted == earlier) {  // all of them
    for (int p = kAll ? threadIdx.x : lane; p < budget; p += kAll ? kWave * kSelectWaves : kWave) out[p] = p <= own ? p : -1;
    return;
  }
  if (wanted == 0) {  // a budget of one page
    if ((kAll ? threadIdx.x : lane) == 0) out[0] = own;
    return;
  }
  uint32_t held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int p = base + k * kWave + lane;
    held[k] = p < earlier ? score_order(scores[p]) : 0;
  }
  int reach;
  const uint32_t least = least_order<kAll, kAll ? kHeld <= 4 ? 3 : 2 : 1>(wanted, earlier, reach, shared, turn, [&](uint32_t number) {
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) mine += __popcll(__ballot(held[k] >= number));
    return mine;
  });
  // those at it are too many by reach - wanted: the first of them are taken
  int at = 0, taken = 0, before_at = 0, before = 0;
  const int spare = reach - wanted;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) at += __popcll(__ballot(held[k] == least));
  const int all_at = count_all<kAll>(at, shared, turn), left = all_at - spare;
  if constexpr (kAll) {
    const uint4* const of = shared + ((turn - 1) & 1) * kSelectWaves;
    for (int w = 0; w < wave; ++w) before_at += of[w].x;
    const int mine_at = left - before_at < 0 ? 0 : left - before_at < at ? left - before_at : at;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) taken += __popcll(__ballot(held[k] > least));
    count_all<kAll>(taken + mine_at, shared, turn);
    const uint4* const now = shared + ((turn - 1) & 1) * kSelectWaves;
    for (int w = 0; w < wave; ++w) before += now[w].x;
  }
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const uint64_t ties = __ballot(held[k] == least);
    const bool take = held[k] > least || (held[k] == least && before_at + static_cast<int>(__popcll(ties & below)) < left);
    before_at += __popcll(ties);
    const uint64_t lanes = __ballot(take);
    if (take) out[before + __popcll(lanes & below)] = base + k * kWave + lane;
    before += __popcll(lanes);
  }
  if ((kAll ? threadIdx.x : lane) == 0) out[wanted] = own;
  for (int p = wanted + 1 + (kAll ? threadIdx.x : lane); p < budget; p += kAll ? kWave * kSelectWaves : kWave) out[p] = -1;
}

// One workgroup per K/V head and `tokens` rows: scores in LDS, then the rows' pages.
template <bool kBf16, int kDim>
__global__ __launch_bounds__(kWave* kSelectWaves) void cache_select_kernel(CacheSelect a, int tokens, int columns) {
  extern __shared__ float scores[];  // [tokens, table_width]
  __shared__ uint4 shared[kCountWords];
  const int wave = threadIdx.x / kWave;
  const int64_t blocks = (a.rows.tokens + tokens - 1) / tokens;
  const int first = static_cast<int>(blockIdx.x % blocks) * tokens;
  const int64_t unit = blockIdx.x / blocks, b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int mine = a.rows.tokens - first < tokens ? a.rows.tokens - first : tokens;
  int most = 0;
  for (int t = 0; t < mine; ++t) {
    const int own = own_page(a, b, first + t);
    most = own > most ? own : most;
  }
  const int width = a.rows.table_width;
  if (a.budget > 1 && most >= a.budget)  // else every page is taken
    for (int from = 0, per = 16 / columns; from < mine; from += per)
      score_pages<kBf16, kDim>(a, b, h, first + from, mine - from < per ? mine - from : per, columns, 16 * wave, most, 16 * kSelectWaves,
                               [&](int token, int page, float score) { scores[(from + token) * width + page] = score; });
  __syncthreads();
  int turn = 0;
  int32_t* const out = a.output + (unit * a.rows.tokens + first) * a.budget;
  if (mine > 1 && most <= kWaveScores) {
    for (int t = wave; t < mine; t += kSelectWaves) {
      const int own = own_page(a, b, first + t);
      if (own <= kWaveScores / 4)
        pick_pages<false, kWaveScores / 4 / kWave>(scores + t * width, own, a.budget, out + static_cast<int64_t>(t) * a.budget, shared, turn);
      else
        pick_pages<false, kWaveScores / kWave>(scores + t * width, own, a.budget, out + static_cast<int64_t>(t) * a.budget, shared, turn);
    }
    return;
  }
  for (int t = 0; t < mine; ++t) {
    const int own = own_page(a, b, first + t);
    if (own <= 4 * kWave * kSelectWaves)
      pick_pages<true, 4>(scores + t * width, own, a.budget, out + static_cast<int64_t>(t) * a.budget, shared, turn);
    else
      pick_pages<true, kRowScores / (kWave * kSelectWaves)>(scores + t * width, own, a.budget, out + static_cast<int64_t>(t) * a.budget, shared, turn);
  }
}

// Short tables: a wave for `tokens` rows, alone.
template <bool kBf16, int kDim>
__global__ __launch_bounds__(kWave* kShortWaves) void cache_select_short_kernel(CacheSelect a, int tokens, int columns) {
  extern __shared__ float scores[];  // [kShortWaves, tokens, table_width]
  const int wave = threadIdx.x / kWave, per_block = tokens * kShortWaves;
  const int64_t blocks = (a.rows.tokens + per_block - 1) / per_block;
  const int first = static_cast<int>(blockIdx.x % blocks) * per_block + wave * tokens;
  const int64_t unit = blockIdx.x / blocks, b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int mine = a.rows.tokens - first < tokens ? a.rows.tokens - first : tokens;
  int most = 0;
  for (int t = 0; t < mine; ++t) {
    const int own = own_page(a, b, first + t);
    most = own > most ? own : most;
  }
  const int width = a.rows.table_width;
  float* const held = scores + static_cast<int64_t>(wave) * tokens * width;
  if (a.budget > 1 && most >= a.budget)  // else every page is taken
    score_pages<kBf16, kDim>(a, b, h, first, mine, columns, 0, most, 16, [&](int token, int page, float score) { held[token * width + page] = score; });
  __threadfence_block();
  int turn = 0;
  int32_t* const out = a.output + (unit * a.rows.tokens + first) * a.budget;
  for (int t = 0; t < mine; ++t)
    pick_pages<false, kShortPages / kWave>(held + t * width, own_page(a, b, first + t), a.budget, out + static_cast<int64_t>(t) * a.budget, nullptr, turn);
}

// Longer tables, and few rows of long ones: scores in the workspace, by as many workgroups as there are pages for ...
constexpr int kScoreTiles = 4;  // of 16 pages, a wave

template <bool kBf16, int kDim>
__global__ __launch_bounds__(256) void cache_score_kernel(CacheSelect a, int columns, int parts) {
  const int64_t row = blockIdx.x / parts;
  const int64_t i = row % a.rows.tokens, unit = row / a.rows.tokens;
  const int64_t b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int own = own_page(a, b, i);
  const int from = static_cast<int>(blockIdx.x % parts) * (4 * kScoreTiles * 16) + threadIdx.x / kWave * (kScoreTiles * 16);
  const int to = own < from + kScoreTiles * 16 ? own : from + kScoreTiles * 16;
  float* const scores = a.scores + row * a.rows.table_width;
  if (own >= a.budget)
    score_pages<kBf16, kDim>(a, b, h, static_cast<int>(i), 1, columns, from, to, 16, [&](int, int page, float score) { scores[page] = score; });
}

// ... and the row's pages from there: from registers, or where they do not hold them by counting in memory.
__global__ __launch_bounds__(kWave* kSelectWaves) void cache_pick_kernel(CacheSelect a) {
  __shared__ uint4 shared[kCountWords];
  const int64_t row = blockIdx.x;
  const int64_t i = row % a.rows.tokens, b = row / a.rows.tokens / a.cache.kv_heads;
  const int own = own_page(a, b, i);
  int32_t* const out = a.output + row * a.budget;
  const float* const scores = a.scores + row * a.rows.table_width;
  int turn = 0;
  if (own <= 4 * kWave * kSelectWaves) {
    pick_pages<true, 4>(scores, own, a.budget, out, shared, turn);
    return;
  }
  if (own <= kRowScores || a.budget > own) {
    pick_pages<true, kRowScores / (kWave * kSelectWaves)>(scores, own, a.budget, out, shared, turn);
    return;
  }
  const int wanted = a.budget - 1;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  // a row of 2^24 pages has counts over 16 bits: one at a time
  const auto count = [&](auto holds) {
    int mine = 0;
    for (int base = wave * kWave; base < own; base += kWave * kSelectWaves) {
      const int p = base + lane;
      mine += __popcll(__ballot(p < own && holds(score_order(scores[p < own ? p : 0]))));
    }
    return mine;
  };
  int reach;
  const uint32_t least = least_order<true, 1>(wanted, own, reach, shared, turn,
                                              [&](uint32_t number) { return static_cast<uint32_t>(count([&](uint32_t u) { return u >= number; })); });
  const int left = count_all<true>(count([&](uint32_t u) { return u == least; }), shared, turn) - (reach - wanted);
  int done = 0, at_done = 0;
  const uint64_t below = (1ull << lane) - 1;
  for (int base = 0; base < own; base += kWave * kSelectWaves) {
    const int p = base + static_cast<int>(threadIdx.x);
    const uint32_t u = p < own ? score_order(scores[p]) : 0;
    const uint64_t ties = __ballot(u == least && p < own);
    const int all_ties = count_all<true>(__popcll(ties), shared, turn);
    int rank = at_done + __popcll(ties & below);
    for (int w = 0; w < wave; ++w) rank += shared[((turn - 1) & 1) * kSelectWaves + w].x;
    at_done += all_ties;
    const bool take = p < own && (u > least || (u == least && rank < left));
    const uint64_t lanes = __ballot(take);
    const int all_taken = count_all<true>(__popcll(lanes), shared, turn);
    int place = done + __popcll(lanes & below);
    for (int w = 0; w < wave; ++w) place += shared[((turn - 1) & 1) * kSelectWaves + w].x;
    if (take) out[place] = p;
    done += all_taken;
  }
  if (threadIdx.x == 0) out[wanted] = own;
}

}  // namespace

// A workgroup for each page that a sequence's rows can touch.
static dim3 move_blocks(const CacheMove& a) {
  return dim3(static_cast<uint32_t>(static_cast<int64_t>(a.batch) * a.cache.kv_heads * pages_touched(a.rows.tokens)));
}

hipError_t launch_cache_write(const CacheMove& a, CacheForm form, hipStream_t stream) {
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    cache_write_kernel<decltype(bf16)::value, decltype(fp8)::value, decltype(dim)::value>
        <<<move_blocks(a), dim3(kWave * kMoveWaves), 0, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_cache_read(const CacheMove& a, CacheForm form, hipStream_t stream) {
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    cache_read_kernel<decltype(bf16)::value, decltype(fp8)::value, decltype(dim)::value>
        <<<move_blocks(a), dim3(kWave * kMoveWaves), 0, stream>>>(a);
    return hipGetLastError();
  });
}

// Columns of a token in a score tile: its heads, up to 16, filled up to a power of two.
static int select_columns(const CacheSelect& a) {
  const int group = a.heads / a.cache.kv_heads;
  int columns = 1;
  while (columns < group && columns < 16) columns *= 2;
  return columns;
}

// Rows of a workgroup whose scores fit its LDS; 0: scores go to the workspace.  That is also the quicker way where there
// are no more rows than CUs and each has over kSplitPages pages: one workgroup reads a row's bounds at what one CU
// gets of the memory's rate.  128 rows of 768 pages took 30.1 us in one kernel, 26.5 in two; of 512 23.8 and 24.1, of 256
// 21.7 and 22.3.
constexpr int kSplitPages = 512;

static int select_tokens(const CacheSelect& a, int cus) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.cache.kv_heads * a.rows.tokens;
  if (a.rows.table_width > kRowScores || (rows <= cus && a.rows.table_width > kSplitPages)) return 0;
  int tokens = std::min(std::min(16 / select_columns(a), kRowScores / a.rows.table_width), a.rows.tokens);
  // A tile's rows; or more, so that each wave picks a row's pages, where a wave holds a row's scores and two workgroups a
  // CU remain.  5664 rows of 16 heads and 258 pages, a row a workgroup, took 290 us, eight a workgroup 207.
  while (a.rows.table_width > kShortPages && a.rows.table_width <= kWaveScores && 2 * tokens <= kSelectWaves &&
         2 * tokens * a.rows.table_width <= kRowScores && rows / (2 * tokens) >= 2 * static_cast<int64_t>(cus))
    tokens *= 2;
  return tokens;
}

int64_t cache_select_scores(const CacheSelect& a, int cus) {
  return select_tokens(a, cus) > 0 ? 0 : static_cast<int64_t>(a.batch) * a.cache.kv_heads * a.rows.tokens * a.rows.table_width;
}

// Whether a wave alone takes its rows: where there are pages for one wave and rows for more.  Eight waves a row's pages
// leave seven without: 56 sequences of 84 rows and up to 9 pages took 51 us, and 16.9 with a wave each; 18 of 64 rows
// and 2 pages 17.4 and 6.1.  At 70 pages (8 sequences of 14 rows) a wave alone took 19 us, eight waves 12.3.
static bool select_short(const CacheSelect& a, int tokens) {
  return tokens > 0 && a.rows.tokens > tokens && a.rows.table_width <= kShortPages;
}

// Workgroups for a row's scores in the workspace.
static int score_parts(const CacheSelect& a) { return static_cast<int>(ceil_div(a.rows.table_width, 4 * kScoreTiles * 16)); }

int64_t cache_select_most_workgroups(const CacheSelect& a) {
  return static_cast<int64_t>(a.batch) * a.cache.kv_heads * a.rows.tokens * score_parts(a);
}

hipError_t launch_cache_select(const CacheSelect& a, CacheForm form, int cus, hipStream_t stream) {
  const int tokens = select_tokens(a, cus), columns = select_columns(a);
  const int64_t units = static_cast<int64_t>(a.batch) * a.cache.kv_heads;
  const dim3 blocks(static_cast<uint32_t>(tokens == 0 ? units * a.rows.tokens * score_parts(a)
                                                      : units * ceil_div(a.rows.tokens, tokens * (select_short(a, tokens) ? kShortWaves : 1))));
  form.fp8 = false;  // the bounds are INT8 in every cache
  return with_cache_form(form, [&](auto bf16, auto, auto dim) {
    constexpr bool kBf16 = decltype(bf16)::value;
    constexpr int kDim = decltype(dim)::value;
    if (select_short(a, tokens)) {
      cache_select_short_kernel<kBf16, kDim>
          <<<blocks, dim3(kWave * kShortWaves), static_cast<size_t>(kShortWaves) * tokens * a.rows.table_width * 4, stream>>>(a, tokens, columns);
      return hipGetLastError();
    }
    if (tokens > 0) {
      cache_select_kernel<kBf16, kDim><<<blocks, dim3(kWave * kSelectWaves), static_cast<size_t>(tokens) * a.rows.table_width * 4, stream>>>(
          a, tokens, columns);
      return hipGetLastError();
    }
    const int parts = score_parts(a);
    cache_score_kernel<kBf16, kDim><<<blocks, dim3(256), 0, stream>>>(a, columns, parts);
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    cache_pick_kernel<<<dim3(blocks.x / parts), dim3(kWave * kSelectWaves), 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace piper

// ---- C entry points --------------------------------------------------------------------------------------------------

namespace {

using piper::aligned16;
using piper::fail;

constexpr int64_t kMaxRows = int64_t(1) << 30;  // of a call, times its heads
constexpr int kMaxThreads = 512;                // of a workgroup of these kernels

int check_version(int32_t version) {
  if (version != PIPER_CACHE_ABI_VERSION)
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "cache ABI version mismatch: caller %d, library %d", version, PIPER_CACHE_ABI_VERSION);
  return PIPER_OK;
}

int check_dtype(int32_t dtype) {
  if (dtype != PIPER_FLOAT16 && dtype != PIPER_BFLOAT16)
    return fail(PIPER_ERROR_UNSUPPORTED, "dtype must be float16 or bfloat16");
  return PIPER_OK;
}

// Sizes of a cache and of a call's rows; no pointer is looked at.
int check_sizes(const piper_cache& c, const piper_cache_rows& r) {
  if (c.head_dim != 64 && c.head_dim != 128) return fail(PIPER_ERROR_UNSUPPORTED, "head_dim must be 64 or 128, got %d", c.head_dim);
  if (c.code != PIPER_CACHE_INT8 && c.code != PIPER_CACHE_FP8) return fail(PIPER_ERROR_UNSUPPORTED, "unknown cache code %d", c.code);
  if (c.pages <= 0 || c.kv_heads <= 0 || r.batch <= 0 || r.tokens <= 0 || r.table_width <= 0)
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "sizes must be positive, got pages=%lld kv_heads=%lld batch=%lld tokens=%lld table_width=%lld",
                (long long)c.pages, (long long)c.kv_heads, (long long)r.batch, (long long)r.tokens, (long long)r.table_width);
  // pages and widths are int32 in the kernels, as table entries are
  if (c.pages > INT32_MAX || r.table_width > (1 << 24) || r.tokens > (1 << 26) || c.kv_heads > (1 << 16) || r.batch > (1 << 24) ||
      r.batch * c.kv_heads > kMaxRows / r.tokens)
    return fail(PIPER_ERROR_UNSUPPORTED, "cache call too large for this build");
  return PIPER_OK;
}

// A launch's threads are counted in 32 bits.
int check_launch(int64_t workgroups) {
  if (workgroups > UINT32_MAX / kMaxThreads) return fail(PIPER_ERROR_UNSUPPORTED, "cache call too large for this build");
  return PIPER_OK;
}

// Workgroups of a write or a read.
int64_t move_workgroups(const piper_cache& c, const piper_cache_rows& r) { return r.batch * c.kv_heads * piper::pages_touched(r.tokens); }

int check_rows(const piper_cache_rows& r) {
  if (r.page_table == nullptr || r.starts == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "page_table or starts is NULL");
  if (r.batch > 1 && r.table_stride < 0) return fail(PIPER_ERROR_INVALID_ARGUMENT, "table_stride must not be negative");
  return PIPER_OK;
}

int check_codes(const piper_cache& c) {
  if (!c.key || !c.key_scale || !c.value || !c.value_scale) return fail(PIPER_ERROR_INVALID_ARGUMENT, "a cache pointer is NULL");
  if (!aligned16(c.key) || !aligned16(c.key_scale) || !aligned16(c.value) || !aligned16(c.value_scale))
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "cache arrays must be 16-byte aligned");
  return PIPER_OK;
}

int check_bounds(const piper_cache& c) {
  if (!c.bounds || !c.bound_scale) return fail(PIPER_ERROR_INVALID_ARGUMENT, "a cache pointer is NULL");
  if (!aligned16(c.bounds)) return fail(PIPER_ERROR_INVALID_ARGUMENT, "cache arrays must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(c.bound_scale) % 4 != 0) return fail(PIPER_ERROR_INVALID_ARGUMENT, "bound_scale must be 4-byte aligned");
  return PIPER_OK;
}

int check_tensor(const char* name, const piper_tensor& t) {
  if (t.data == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "%s pointer is NULL", name);
  if (!aligned16(t.data) || t.stride_batch % 8 != 0 || t.stride_head % 8 != 0 || t.stride_seq % 8 != 0)
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "%s must be 16-byte aligned with strides that are multiples of 8 elements", name);
  return PIPER_OK;
}

int check_output(const char* name, const void* p) {
  if (p == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "%s pointer is NULL", name);
  if (!aligned16(p)) return fail(PIPER_ERROR_INVALID_ARGUMENT, "%s must be 16-byte aligned", name);
  return PIPER_OK;
}

int check_heads(int64_t heads, const piper_cache& c, const piper_cache_rows& r) {
  if (heads <= 0 || heads % c.kv_heads != 0)
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "heads must be a positive multiple of kv_heads, got %lld and %lld", (long long)heads,
                (long long)c.kv_heads);
  if (heads > (1 << 20) || r.batch * heads > kMaxRows / r.tokens) return fail(PIPER_ERROR_UNSUPPORTED, "cache call too large for this build");
  return PIPER_OK;
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
  if (need == 0) return PIPER_OK;
  if (workspace == nullptr || bytes < need)
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "the call needs a workspace of %lld bytes, got %lld", (long long)need, (long long)bytes);
  if (!aligned16(workspace)) return fail(PIPER_ERROR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  return PIPER_OK;
}

int launched(hipError_t err, const char* what) {
  return err == hipSuccess ? PIPER_OK : fail(PIPER_ERROR_HIP, "%s launch failed: %s", what, hipGetErrorString(err));
}

piper::Cache cache_of(const piper_cache& c) {
  return piper::Cache{static_cast<uint8_t*>(c.key), c.key_scale, static_cast<uint8_t*>(c.value), c.value_scale, c.bounds, c.bound_scale,
                      static_cast<int32_t>(c.kv_heads)};
}

piper::CacheRows rows_of(const piper_cache& c, const piper_cache_rows& r) {
  return piper::CacheRows{r.page_table, r.starts, r.counts, r.table_stride, c.pages, static_cast<int32_t>(r.table_width),
                          static_cast<int32_t>(r.tokens)};
}

piper::InputTensor input_of(const piper_tensor& t) {
  return piper::InputTensor{t.data, static_cast<long>(t.stride_batch), static_cast<long>(t.stride_head), static_cast<long>(t.stride_seq)};
}

piper::CacheForm form_of(const piper_cache& c, int32_t dtype) {
  return piper::CacheForm{dtype == PIPER_BFLOAT16, c.code == PIPER_CACHE_FP8, c.head_dim};
}

int check_attention(const piper_cache_attention_args* a) {
  if (a == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "args is NULL");
  if (int st = check_version(a->abi_version)) return st;
  if (int st = check_dtype(a->dtype)) return st;
  if (int st = check_sizes(a->cache, a->rows)) return st;
  if (int st = check_heads(a->heads, a->cache, a->rows)) return st;
  if (a->selected != nullptr && (a->budget <= 0 || a->budget > (1 << 24)))
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "budget must be positive, got %lld", (long long)a->budget);
  if (a->selected != nullptr && a->mask != nullptr)
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "a mask and selected pages do not go together");
  return PIPER_OK;
}

piper::CacheAttention attention_of(const piper_cache_attention_args& a) {
  return piper::CacheAttention{cache_of(a.cache), rows_of(a.cache, a.rows), input_of(a.query), a.mask, a.mask_stride_batch,
                               a.mask_stride_row, a.selected, a.output, a.scale, static_cast<int32_t>(a.rows.batch),
                               static_cast<int32_t>(a.heads), static_cast<int32_t>(a.selected != nullptr ? a.budget : 0),
                               piper::CacheShares::kWhole, 1, 1, 1, 1, nullptr, nullptr, nullptr};
}

int check_select(const piper_cache_select_args* a) {
  if (a == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "args is NULL");
  if (int st = check_version(a->abi_version)) return st;
  if (int st = check_dtype(a->dtype)) return st;
  if (int st = check_sizes(a->cache, a->rows)) return st;
  if (int st = check_heads(a->heads, a->cache, a->rows)) return st;
  if (a->budget <= 0 || a->budget > (1 << 24)) return fail(PIPER_ERROR_INVALID_ARGUMENT, "budget must be positive, got %lld", (long long)a->budget);
  return PIPER_OK;
}

piper::CacheSelect select_of(const piper_cache_select_args& a) {
  return piper::CacheSelect{cache_of(a.cache), rows_of(a.cache, a.rows), input_of(a.query), a.output, static_cast<float*>(a.workspace),
                            static_cast<int32_t>(a.rows.batch), static_cast<int32_t>(a.heads), static_cast<int32_t>(a.budget)};
}

}  // namespace

extern "C" int piper_cache_abi_version(void) { return PIPER_CACHE_ABI_VERSION; }

extern "C" int piper_cache_write(const piper_cache_write_args* a, void* stream) {
  if (a == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "args is NULL");
  if (int st = check_version(a->abi_version)) return st;
  if (int st = check_dtype(a->dtype)) return st;
  if (int st = check_sizes(a->cache, a->rows)) return st;
  if (int st = check_launch(move_workgroups(a->cache, a->rows))) return st;
  if (int st = check_rows(a->rows)) return st;
  if (int st = check_codes(a->cache)) return st;
  if (int st = check_bounds(a->cache)) return st;
  if (int st = check_tensor("key", a->key)) return st;
  if (int st = check_tensor("value", a->value)) return st;
  const piper::CacheMove move{cache_of(a->cache), rows_of(a->cache, a->rows), input_of(a->key), input_of(a->value),
                              static_cast<int32_t>(a->rows.batch)};
  return launched(piper::launch_cache_write(move, form_of(a->cache, a->dtype), static_cast<hipStream_t>(stream)), "cache write");
}

extern "C" int piper_cache_read(const piper_cache_read_args* a, void* stream) {
  if (a == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "args is NULL");
  if (int st = check_version(a->abi_version)) return st;
  if (int st = check_dtype(a->dtype)) return st;
  if (int st = check_sizes(a->cache, a->rows)) return st;
  if (int st = check_launch(move_workgroups(a->cache, a->rows))) return st;
  if (int st = check_rows(a->rows)) return st;
  if (int st = check_codes(a->cache)) return st;
  if (int st = check_output("key", a->key)) return st;
  if (int st = check_output("value", a->value)) return st;
  const piper::CacheMove move{cache_of(a->cache), rows_of(a->cache, a->rows), piper::InputTensor{a->key, 0, 0, 0},
                              piper::InputTensor{a->value, 0, 0, 0}, static_cast<int32_t>(a->rows.batch)};
  return launched(piper::launch_cache_read(move, form_of(a->cache, a->dtype), static_cast<hipStream_t>(stream)), "cache read");
}

extern "C" int piper_cache_attention_workspace_bytes(const piper_cache_attention_args* a, int64_t* bytes) {
  if (bytes == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "bytes is NULL");
  if (int st = check_attention(a)) return st;
  int cus = 0, xccs = 0;
  if (int st = piper::device_topology(&cus, &xccs)) return st;
  const piper::CacheParts parts = piper::cache_attention_parts(attention_of(*a), a->cache.head_dim, cus);
  if (int st = check_launch(parts.workgroups)) return st;
  *bytes = parts.bytes;
  return PIPER_OK;
}

extern "C" int piper_cache_attention(const piper_cache_attention_args* a, void* stream) {
  if (int st = check_attention(a)) return st;
  if (!(std::isfinite(a->scale) && a->scale > 0.0f)) return fail(PIPER_ERROR_INVALID_ARGUMENT, "scale must be finite and positive");
  if (int st = check_rows(a->rows)) return st;
  if (int st = check_codes(a->cache)) return st;
  if (int st = check_tensor("query", a->query)) return st;
  if (int st = check_output("output", a->output)) return st;
  if (a->mask != nullptr && (a->mask_stride_batch < 0 || a->mask_stride_row < 0))
    return fail(PIPER_ERROR_INVALID_ARGUMENT, "mask strides must not be negative");
  int cus = 0, xccs = 0;
  if (int st = piper::device_topology(&cus, &xccs)) return st;
  piper::CacheAttention attention = attention_of(*a);
  const piper::CacheParts parts = piper::cache_attention_parts(attention, a->cache.head_dim, cus);
  if (int st = check_launch(parts.workgroups)) return st;  // more than there are to join
  if (int st = check_workspace(a->workspace, a->workspace_bytes, parts.bytes)) return st;
  attention.shares = parts.shares;
  attention.parts = static_cast<int32_t>(parts.parts);
  attention.blocks_of_unit = static_cast<int32_t>(parts.blocks_of_unit);
  attention.least_share = static_cast<int32_t>(parts.least_share);
  attention.workgroups = parts.workgroups;
  attention.partial = static_cast<float*>(a->workspace);
  attention.partial_stats = reinterpret_cast<float2*>(attention.partial + parts.rows * a->cache.head_dim);
  attention.pieces = reinterpret_cast<piper::CachePieces*>(attention.partial_stats + parts.rows);
  return launched(piper::launch_cache_attention(attention, form_of(a->cache, a->dtype), static_cast<hipStream_t>(stream)),
                  "cache attention");
}

extern "C" int piper_cache_select_workspace_bytes(const piper_cache_select_args* a, int64_t* bytes) {
  if (bytes == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "bytes is NULL");
  if (int st = check_select(a)) return st;
  int cus = 0, xccs = 0;
  if (int st = piper::device_topology(&cus, &xccs)) return st;
  const piper::CacheSelect select = select_of(*a);
  if (int st = check_launch(piper::cache_select_most_workgroups(select))) return st;
  *bytes = 4 * piper::cache_select_scores(select, cus);
  return PIPER_OK;
}

extern "C" int piper_cache_select(const piper_cache_select_args* a, void* stream) {
  if (int st = check_select(a)) return st;
  if (int st = check_rows(a->rows)) return st;
  if (int st = check_bounds(a->cache)) return st;
  if (int st = check_tensor("query", a->query)) return st;
  if (a->output == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "output pointer is NULL");
  const piper::CacheSelect select = select_of(*a);
  int cus = 0, xccs = 0;
  if (int st = piper::device_topology(&cus, &xccs)) return st;
  if (int st = check_launch(piper::cache_select_most_workgroups(select))) return st;
  if (int st = check_workspace(a->workspace, a->workspace_bytes, 4 * piper::cache_select_scores(select, cus))) return st;
  return launched(piper::launch_cache_select(select, form_of(a->cache, a->dtype), cus, static_cast<hipStream_t>(stream)), "cache select");
}
