// Attention over the quantised paged cache (include/piper_cache.h).
//
// A call's units are the (sequence, K/V head) pairs, or with selected pages the (sequence, K/V head, token) triples.
// A unit's rows are its query heads' rows, token by token: r = t * group + g.
#include <type_traits>

#include "cache_kernels.h"
#include "host.h"

namespace piper {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;  // of a workgroup: each takes every fourth page
constexpr float kNone = -__builtin_inff();

// Four code bytes as four exact halves.  INT8: the byte with its sign bit flipped is code + 128; under the exponent
// of 1024 it reads as 1024 + 128 + code, and the subtraction is exact.
template <bool kFp8>
__device__ __forceinline__ uint2 halves_of(uint32_t codes) {
  if constexpr (kFp8) {
    return uint2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true))};
  } else {
    const uint32_t u = codes ^ 0x80808080u;
    const half2_t offset = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const half2_t lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + offset;
    const half2_t hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + offset;
    return uint2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
}

template <bool kFp8>
__device__ __forceinline__ half8 halves_of(uint32_t lo, uint32_t hi) {
  const uint2 a = halves_of<kFp8>(lo), b = halves_of<kFp8>(hi);
  return __builtin_bit_cast(half8, uint4{a.x, a.y, b.x, b.y});
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Max / sum over the four lanes that hold a column of a 16x16 result (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return cross_half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

__device__ __forceinline__ float column_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return cross_half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// The pages of a unit and how they are split: `parts` equal ranges, one workgroup each.
struct PageRange {
  int pages, parts;
};

__device__ __forceinline__ PageRange page_range(const CacheAttention& a, int64_t b) {
  const int count = a.rows.count(b);
  const int pages = a.selected != nullptr ? a.budget : static_cast<int>((count > 0 ? a.rows.end(b, count - 1) + kPage - 1 : 0) / kPage);
  const int parts = (pages + a.part_pages - 1) / a.part_pages;
  return PageRange{pages, parts < 1 ? 1 : parts > a.parts ? a.parts : parts};
}

// One workgroup per unit, block of 16 kTiles rows and part of the pages.  K and V go from memory to the matrix
// instructions' operands in registers: S^T = K Q^T and O^T = V^T P^T, so a lane's scores are already the P that it
// has to give, and the cache's layouts are such that 16 consecutive bytes are a lane's operand.
//   K: lane (m, g) = (lane % 16, lane / 16) takes 16 bytes of row key(m), features 64 c + 16 g on.  Row m of tile t in
//      half hh is key 32 hh + 8 (m / 4) + 4 t + m % 4: then column n's lane (n, g) holds keys 32 hh + 8 g + 0..7.
//   V: lane (m, g) takes 16 bytes: keys 32 hh + 8 g + 0..7 of features 32 f + 2 m and 32 f + 2 m + 1.
template <bool kBf16, bool kFp8, int kDim, int kTiles>
struct Stream {
  static constexpr int kChunks = kDim / 64, kFeatures = kDim / 32;  // K pieces of a row; pairs of V tiles
  const CacheAttention& a;
  int lane, n, g;
  half8 query[kTiles][kChunks][2];
  float factor[kTiles];            // scores in powers of two: accumulator * key scale * factor
  float top[kTiles], total[kTiles];  // the running maximum; this lane's share of the sum
  float4_t sum[kTiles][2 * kFeatures];
  float reference;  // a power of two no value scale so far is above: sums hold 2^15 / reference times the values
  uint4 key[2][2][kChunks], value[2][kFeatures];
  float4 key_scale[2][2], value_scale[2][2];

  __device__ __forceinline__ explicit Stream(const CacheAttention& args) : a(args) {
    lane = threadIdx.x % kWave;
    n = lane % 16;
    g = lane / 16;
    reference = 0x1p-100f;
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
      top[r] = kNone;
      total[r] = 0.0f;
#pragma unroll
      for (int f = 0; f < 2 * kFeatures; ++f) sum[r][f] = float4_t{0, 0, 0, 0};
    }
  }

  // A row of the query as halves scaled by the power of two that brings its largest value near 2^15: exact for
  // FP16 and BF16 down to 2^-29 of that value (smaller ones become subnormal or vanish).
  __device__ __forceinline__ void load_query(int r, const uint16_t* row) {
    uint4 raw[kChunks][2];
    float x[8], largest = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        raw[c][e] = row != nullptr ? *reinterpret_cast<const uint4*>(row + 64 * c + 16 * g + 8 * e) : uint4{0, 0, 0, 0};
        widen8<kBf16>(raw[c][e], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
      }
    const int exponent = static_cast<int>(__float_as_uint(column_max(largest)) >> 23);  // biased
    const int up = 268 - exponent > 254 ? 254 : 268 - exponent;
    const float scale = __uint_as_float(static_cast<uint32_t>(up) << 23);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        widen8<kBf16>(raw[c][e], x);
        uint4 packed;
        packed.x = pack_half2(x[0] * scale, x[1] * scale);
        packed.y = pack_half2(x[2] * scale, x[3] * scale);
        packed.z = pack_half2(x[4] * scale, x[5] * scale);
        packed.w = pack_half2(x[6] * scale, x[7] * scale);
        query[r][c][e] = __builtin_bit_cast(half8, packed);
      }
    factor[r] = a.scale * kLog2e / scale;
  }

  __device__ __forceinline__ void load_key(int64_t record) {
    const uint8_t* const k = a.cache.key + record * (kPage * kDim) + (8 * (n / 4) + n % 4) * kDim + 16 * g;
    const float* const s = a.cache.key_scale + record * kPage + 8 * g;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) key[hh][t][c] = *reinterpret_cast<const uint4*>(k + (32 * hh + 4 * t) * kDim + 64 * c);
        key_scale[hh][t] = *reinterpret_cast<const float4*>(s + 32 * hh + 4 * t);
      }
  }

  __device__ __forceinline__ void load_value(int64_t record) {
    const uint8_t* const v = a.cache.value + record * (kPage * kDim) + g * (8 * kDim) + 16 * n;
    const float* const s = a.cache.value_scale + record * kPage + 8 * g;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
      for (int f = 0; f < kFeatures; ++f) value[hh][f] = *reinterpret_cast<const uint4*>(v + hh * (32 * kDim) + f * 256);
#pragma unroll
      for (int t = 0; t < 2; ++t) value_scale[hh][t] = *reinterpret_cast<const float4*>(s + 32 * hh + 4 * t);
    }
  }

  // S^T of the loaded page times the key scales: score[r][hh][t][i] is key 32 hh + 8 g + 4 t + i of row n.
  __device__ __forceinline__ void scores(float4_t (&score)[kTiles][2][2]) const {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < kTiles; ++r) score[r][hh][t] = float4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const half8 lo = halves_of<kFp8>(key[hh][t][c].x, key[hh][t][c].y), hi = halves_of<kFp8>(key[hh][t][c].z, key[hh][t][c].w);
#pragma unroll
          for (int r = 0; r < kTiles; ++r) {
            score[r][hh][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, query[r][c][0], score[r][hh][t], 0, 0, 0);
            score[r][hh][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, query[r][c][1], score[r][hh][t], 0, 0, 0);
          }
        }
        const float4 s = key_scale[hh][t];
#pragma unroll
        for (int r = 0; r < kTiles; ++r) score[r][hh][t] *= float4_t{s.x, s.y, s.z, s.w};
      }
  }

  // The softmax's weights of a page and its share of the sums.  `visible(r, key)` with kMasked; `keys`: slots of the
  // page from here on hold nothing that any row sees.
  template <bool kMasked, typename Visible>
  __device__ __forceinline__ void accumulate(float4_t (&score)[kTiles][2][2], int keys, Visible visible) {
    float scales[2][2][4], largest = 0.0f;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float s[4] = {value_scale[hh][t].x, value_scale[hh][t].y, value_scale[hh][t].z, value_scale[hh][t].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          scales[hh][t][i] = kMasked && 32 * hh + 8 * g + 4 * t + i >= keys ? 0.0f : s[i];
          largest = fmaxf(largest, scales[hh][t][i]);
        }
      }
    largest = column_max(largest);
    const float above = __uint_as_float((__float_as_uint(largest) & 0x7f800000u) + 0x00800000u);
    const float next_reference = fmaxf(reference, above);
    const float shrink = reference / next_reference;
    bool changed = next_reference > reference;
    reference = next_reference;
    const float unit = 0x1p15f / reference;

    half8 weight[kTiles][2];
    float keep[kTiles];
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
      float page_top = kNone;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (kMasked)
              if (!visible(r, 32 * hh + 8 * g + 4 * t + i)) score[r][hh][t][i] = kNone;
            page_top = fmaxf(page_top, score[r][hh][t][i]);
          }
      const float next = fmaxf(top[r], column_max(page_top) * factor[r]);
      const float base = next == kNone ? 0.0f : next;
      keep[r] = exp2_fast(top[r] - base);
      changed = changed || next > top[r];
      top[r] = next;
      total[r] *= keep[r];
      keep[r] *= shrink;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t packed[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float s = score[r][hh][t][i];
            // an unseen key's score is -inf, also times the factor; its value scale may be anything
            const float p = exp2_fast(fmaf(s, factor[r], -base));
            total[r] += p;
            w[i] = p * (scales[hh][t][i] * unit);
            if constexpr (kMasked) w[i] = s == kNone ? 0.0f : w[i];
          }
          packed[2 * t] = pack_half2(w[0], w[1]);
          packed[2 * t + 1] = pack_half2(w[2], w[3]);
        }
        weight[r][hh] = __builtin_bit_cast(half8, uint4{packed[0], packed[1], packed[2], packed[3]});
      }
    }
    if (__any(changed)) {
#pragma unroll
      for (int r = 0; r < kTiles; ++r)
#pragma unroll
        for (int f = 0; f < 2 * kFeatures; ++f) sum[r][f] *= keep[r];
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      // codes of slots that hold nothing could be FP8 NaN, which zero weights do not cancel
      const int held = keys - 32 * hh - 8 * g;
      const uint32_t low = held >= 4 ? ~0u : held <= 0 ? 0u : (1u << (8 * held)) - 1;
      const uint32_t high = held >= 8 ? ~0u : held <= 4 ? 0u : (1u << (8 * (held - 4))) - 1;
#pragma unroll
      for (int f = 0; f < kFeatures; ++f) {
        uint4 v = value[hh][f];
        if constexpr (kMasked && kFp8) v = uint4{v.x & low, v.y & high, v.z & low, v.w & high};
        const half8 even = halves_of<kFp8>(v.x, v.y), odd = halves_of<kFp8>(v.z, v.w);
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          sum[r][2 * f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, weight[r][hh], sum[r][2 * f], 0, 0, 0);
          sum[r][2 * f + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, weight[r][hh], sum[r][2 * f + 1], 0, 0, 0);
        }
      }
    }
  }
};

template <bool kBf16, bool kFp8, int kDim, int kTiles>
__global__ __launch_bounds__(kWave* kWaves, kTiles == 1 ? 2 : 1) void cache_stream_kernel(CacheAttention a) {
  constexpr int kRows = 16 * kTiles, kPad = kDim + 4;
  __shared__ float shared_sum[kWaves][16][kPad];
  __shared__ float shared_top[kWaves][16], shared_total[kWaves][16];
  const int wave = threadIdx.x / kWave;
  const int group = a.heads / a.cache.kv_heads;
  const int unit_tokens = a.selected != nullptr ? 1 : a.rows.tokens;
  const int unit_rows = unit_tokens * group;
  const int blocks = (unit_rows + kRows - 1) / kRows;
  int64_t at = blockIdx.x;
  const int part = static_cast<int>(at % a.parts);
  at /= a.parts;
  const int first_row = static_cast<int>(at % blocks) * kRows;
  const int64_t unit = at / blocks;
  const int first_token = a.selected != nullptr ? static_cast<int>(unit % a.rows.tokens) : 0;
  const int64_t pair = a.selected != nullptr ? unit / a.rows.tokens : unit;
  const int64_t b = pair / a.cache.kv_heads, h = pair % a.cache.kv_heads;
  const PageRange range = page_range(a, b);
  if (part >= range.parts) return;
  const int start = a.rows.starts[b];
  const int count = a.rows.count(b);

  Stream<kBf16, kFp8, kDim, kTiles> s(a);
  int token[kTiles];
  int limit[kTiles];  // what the lane's row of each tile sees stands before this position
  int most = 0, least = 0;  // the largest limit, and what every row with a limit sees stands before
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    const int row = first_row + 16 * r + s.n;
    token[r] = first_token + row / group;
    const bool real = row < unit_rows && token[r] < count;
    const uint16_t* q = static_cast<const uint16_t*>(a.query.data) + b * a.query.stride_batch + (h * group + row % group) * a.query.stride_head +
                        token[r] * a.query.stride_seq;
    s.load_query(r, real ? q : nullptr);
    limit[r] = real ? static_cast<int>(a.rows.end(b, a.mask != nullptr ? count - 1 : token[r])) : 0;
  }
  {
    const int last = first_row + kRows < unit_rows ? first_row + kRows - 1 : unit_rows - 1;
    const int first_t = first_token + first_row / group;
    const int last_t = first_token + last / group < count ? first_token + last / group : count - 1;
    if (first_t < count) {
      most = static_cast<int>(a.rows.end(b, a.mask != nullptr ? count - 1 : last_t));
      least = a.mask != nullptr ? (start < most ? (start > 0 ? start : 0) : most) : static_cast<int>(a.rows.end(b, first_t));
    }
  }

  const int lo = static_cast<int>(static_cast<int64_t>(range.pages) * part / range.parts);
  int hi = static_cast<int>(static_cast<int64_t>(range.pages) * (part + 1) / range.parts);
  const int end_page = (most + kPage - 1) / kPage;
  const int32_t* const selected = a.selected != nullptr ? a.selected + unit * a.budget : nullptr;
  if (selected == nullptr && hi > end_page) hi = end_page;

  // the next page of this wave that the table names, from step `step` on
  const auto find = [&](int& step, int& logical, int64_t& record) {
    for (; step < hi; step += kWaves) {
      logical = __builtin_amdgcn_readfirstlane(selected != nullptr ? selected[step] : step);
      if (logical >= end_page) continue;
      const int64_t page = a.rows.page(b, logical);
      if (page < 0) continue;
      record = page * a.cache.kv_heads + h;
      return true;
    }
    return false;
  };
  int step = lo + __builtin_amdgcn_readfirstlane(wave), logical = 0;
  int64_t record = 0;
  bool more = find(step, logical, record);
  if (more) {
    s.load_key(record);
    s.load_value(record);
  }
  while (more) {
    const int base = logical * kPage;
    step += kWaves;
    more = find(step, logical, record);
    float4_t score[kTiles][2][2];
    s.scores(score);
    if (more) s.load_key(record);
    if (base + kPage <= least) {
      s.template accumulate<false>(score, kPage, [](int, int) { return true; });
    } else {
      const int keys = most - base < kPage ? most - base : kPage;
      s.template accumulate<true>(score, keys, [&](int r, int key) {
        const int position = base + key;
        bool seen = position < limit[r];
        if (a.mask != nullptr && position >= start && seen)
          seen = a.mask[b * a.mask_stride_batch + token[r] * a.mask_stride_row + (position - start)] != 0;
        return seen;
      });
    }
    if (more) s.load_value(record);
  }

  // the waves' sums joined, a row tile at a time: 16 threads a row
  constexpr int kPer = kDim / 16;
  const int row16 = threadIdx.x / 16, piece = threadIdx.x % 16;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens;
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    const float total = column_sum(s.total[r]);
    const float value_unit = s.reference * 0x1p-15f;
    if (r > 0) __syncthreads();
    if (s.g == 0) {
      shared_top[wave][s.n] = s.top[r];
      shared_total[wave][s.n] = total;
    }
#pragma unroll
    for (int f = 0; f < kDim / 32; ++f) {
      const float4_t even = s.sum[r][2 * f], odd = s.sum[r][2 * f + 1];
      float4* const to = reinterpret_cast<float4*>(&shared_sum[wave][s.n][32 * f + 8 * s.g]);
      to[0] = float4{even[0] * value_unit, odd[0] * value_unit, even[1] * value_unit, odd[1] * value_unit};
      to[1] = float4{even[2] * value_unit, odd[2] * value_unit, even[3] * value_unit, odd[3] * value_unit};
    }
    __syncthreads();
    const int row = first_row + 16 * r + row16;
    if (row >= unit_rows) continue;
    float top = kNone;
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, shared_top[w][row16]);
    const float base = top == kNone ? 0.0f : top;
    float joined = 0.0f, x[kPer] = {};
    for (int w = 0; w < kWaves; ++w) {
      const float scale = exp2_fast(shared_top[w][row16] - base);
      joined += shared_total[w][row16] * scale;
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = fmaf(shared_sum[w][row16][piece * kPer + e], scale, x[e]);
    }
    const int t = first_token + row / group;
    if (range.parts > 1) {
      const int64_t at_row = part * rows + (pair * a.rows.tokens * group + (a.selected != nullptr ? t * group + row : row));
      float* const to = a.partial + at_row * kDim + piece * kPer;
#pragma unroll
      for (int e = 0; e < kPer; e += 4) *reinterpret_cast<float4*>(to + e) = float4{x[e], x[e + 1], x[e + 2], x[e + 3]};
      if (piece == 0) a.partial_stats[at_row] = float2{top, joined};
      continue;
    }
    // a row beyond the count has gone through the pages that every real row sees, whatever they hold
    const bool none = joined == 0.0f || t >= count;
    const float inverse = 1.0f / joined;
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = none ? 0.0f : x[e] * inverse;
    uint16_t* const out = static_cast<uint16_t*>(a.output) + ((b * a.heads + h * group + row % group) * a.rows.tokens + t) * kDim + piece * kPer;
#pragma unroll
    for (int e = 0; e < kPer; e += 4)
      *reinterpret_cast<uint2*>(out + e) = uint2{narrow2<kBf16>(x[e], x[e + 1]), narrow2<kBf16>(x[e + 2], x[e + 3])};
  }
}

// The parts' sums joined: one wave per row.
template <bool kBf16, int kDim>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttention a) {
  constexpr int kPer = kDim / kWave;
  const int lane = threadIdx.x % kWave;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (row >= rows) return;
  const int group = a.heads / a.cache.kv_heads;
  const int64_t pair = row / (static_cast<int64_t>(a.rows.tokens) * group), b = pair / a.cache.kv_heads, h = pair % a.cache.kv_heads;
  const int within = static_cast<int>(row % (static_cast<int64_t>(a.rows.tokens) * group)), t = within / group;
  const PageRange range = page_range(a, b);
  if (range.parts == 1) return;
  const int parts = t < a.rows.count(b) ? range.parts : 0;
  float top = kNone;
  for (int p = 0; p < parts; ++p) top = fmaxf(top, a.partial_stats[p * rows + row].x);
  const float base = top == kNone ? 0.0f : top;
  float total = 0.0f, x[kPer] = {};
  for (int p = 0; p < parts; ++p) {
    const float2 stats = a.partial_stats[p * rows + row];
    const float scale = exp2_fast(stats.x - base);
    total = fmaf(stats.y, scale, total);
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = fmaf(a.partial[(p * rows + row) * kDim + lane * kPer + e], scale, x[e]);
  }
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
  uint16_t* const out = static_cast<uint16_t*>(a.output) + ((b * a.heads + h * group + within % group) * a.rows.tokens + t) * kDim + lane * kPer;
  const uint32_t packed = narrow2<kBf16>(x[0] * inverse, x[kPer - 1] * inverse);
  if constexpr (kPer == 2)
    *reinterpret_cast<uint32_t*>(out) = packed;
  else
    *out = static_cast<uint16_t>(packed);
}

}  // namespace

// Rows of a unit, and how many units.
static int64_t unit_rows(const CacheAttention& a) {
  return (a.selected != nullptr ? 1 : static_cast<int64_t>(a.rows.tokens)) * (a.heads / a.cache.kv_heads);
}

static int row_tiles(const CacheAttention& a) { return unit_rows(a) <= 16 ? 1 : 2; }

CacheParts cache_attention_parts(const CacheAttention& a, int head_dim, int cus) {
  const int64_t units = static_cast<int64_t>(a.batch) * a.cache.kv_heads * (a.selected != nullptr ? a.rows.tokens : 1);
  const int64_t blocks = units * ceil_div(unit_rows(a), 16 * row_tiles(a));
  const int64_t pages = a.selected != nullptr ? a.budget : a.rows.table_width;
  // enough workgroups for four rounds of two a CU, none with fewer pages than waves
  const int64_t wanted = ceil_div(8 * static_cast<int64_t>(cus), blocks);
  int64_t part_pages = ceil_div(pages, wanted);
  if (part_pages < kWaves) part_pages = kWaves;
  CacheParts p;
  p.part_pages = static_cast<int32_t>(part_pages);
  p.parts = static_cast<int32_t>(ceil_div(pages, part_pages));
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens;
  p.bytes = p.parts > 1 ? p.parts * rows * (head_dim + 2) * 4 : 0;
  p.stats_offset = p.parts * rows * head_dim * 4;
  p.blocks = blocks * p.parts;
  return p;
}

hipError_t launch_cache_attention(const CacheAttention& a, const CacheParts& parts, CacheForm form, hipStream_t stream) {
  const dim3 blocks(static_cast<uint32_t>(parts.blocks));
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    constexpr bool kBf16 = decltype(bf16)::value, kFp8 = decltype(fp8)::value;
    constexpr int kDim = decltype(dim)::value;
    if (row_tiles(a) == 1)
      cache_stream_kernel<kBf16, kFp8, kDim, 1><<<blocks, dim3(kWave * kWaves), 0, stream>>>(a);
    else
      cache_stream_kernel<kBf16, kFp8, kDim, 2><<<blocks, dim3(kWave * kWaves), 0, stream>>>(a);
    if (const hipError_t err = hipGetLastError(); err != hipSuccess || parts.parts == 1) return err;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens;
    cache_join_kernel<kBf16, kDim><<<dim3(static_cast<uint32_t>(ceil_div(rows, 4))), dim3(256), 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace piper
