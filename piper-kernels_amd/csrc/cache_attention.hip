// Attention over the quantised paged cache (include/piper_cache.h).
//
// A call's units are the (sequence, K/V head) pairs, or with selected pages the (sequence, K/V head, token) triples.
// A unit's rows are its query heads' rows, token by token: r = t * group + g.
#include <algorithm>
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

// Codes that one workgroup alone reads, once: past the caches' replacement order.
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(p)));
}

template <bool kFp8>
__device__ __forceinline__ half8 halves_of(uint32_t lo, uint32_t hi) {
  const uint2 a = halves_of<kFp8>(lo), b = halves_of<kFp8>(hi);
  return __builtin_bit_cast(half8, uint4{a.x, a.y, b.x, b.y});
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The power of two that brings a query row's largest value near 2^15.  Rows of halves so scaled are exact for FP16 and
// BF16 down to 2^-29 of that value (smaller ones become subnormal or vanish).
__device__ __forceinline__ float query_scale(float largest) {
  const int up = 268 - static_cast<int>(__float_as_uint(largest) >> 23);  // biased
  return __uint_as_float(static_cast<uint32_t>(up > 254 ? 254 : up) << 23);
}

template <bool kBf16>
__device__ __forceinline__ half8 scaled_halves(const uint4 raw, float scale) {
  float x[8];
  widen8<kBf16>(raw, x);
  return __builtin_bit_cast(half8, uint4{pack_half2(x[0] * scale, x[1] * scale), pack_half2(x[2] * scale, x[3] * scale),
                                         pack_half2(x[4] * scale, x[5] * scale), pack_half2(x[6] * scale, x[7] * scale)});
}

template <bool kBf16>
__device__ __forceinline__ float largest_of(const uint4 raw, float largest) {
  float x[8];
  widen8<kBf16>(raw, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(x[i]));
  return largest;
}

// Max / sum over the four lanes that hold a column of a 16x16 result (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return cross_half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

__device__ __forceinline__ float column_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return cross_half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ int wave_prefix(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int up = __shfl_up(v, d, kWave);
    if (static_cast<int>(threadIdx.x % kWave) >= d) v += up;
  }
  return v;
}

// Entries of a unit's list up to its last page: what follows that (a list shorter than the budget ends in -1) is not
// walked through.  1584 lists of up to 5 pages in a budget of 102: 244 us with, 22 without; where lists are full, finding
// that out takes 0.2 us.
__device__ __forceinline__ int listed_pages(const CacheAttention& a, int64_t unit) {
  const int32_t* const list = a.selected + unit * a.budget;
  int n = 0;
  for (int from = 0; from < a.budget; from += kWave) {
    const int i = from + static_cast<int>(threadIdx.x % kWave);
    const uint64_t pages = __ballot(i < a.budget && list[i < a.budget ? i : 0] >= 0);
    if (pages != 0) n = from + kWave - __builtin_clzll(pages);
  }
  return n;
}

// Pages of each of a sequence's blocks.
__device__ __forceinline__ int pages_of(const CacheAttention& a, int64_t b) {
  const int count = a.rows.count(b);
  return count > 0 ? static_cast<int>((a.rows.end(b, count - 1) + kPage - 1) / kPage) : 0;
}

// Pages `lo` to `hi` of a block: all of them (`whole`), or a piece whose sums go to the workspace.
struct Piece {
  int64_t b, block;  // sequence, block of its K/V heads' rows
  int lo, hi;
  bool whole;
  int64_t index;  // in the workspace
};

// CacheShares::kLine: the pages of all blocks that have rows stand in one line, sequence by sequence, and workgroup w takes
// the `share` pages from w * share on: parts of two blocks and the blocks between.  So sequences of any lengths give every
// workgroup the same work, and there are no more pieces to join than workgroups.  Calls f(piece) for each block of the
// workgroup.
template <typename F>
__device__ __forceinline__ void walk_line(const CacheAttention& a, int block_rows, F f) {
  const int lane = threadIdx.x % kWave, group = a.heads / a.cache.kv_heads, heads = a.cache.kv_heads;
  const auto blocks_of = [&](int64_t b) { return (a.rows.count(b) * group + block_rows - 1) / block_rows; };  // of a head
  const auto length = [&](int64_t b) { return b < a.batch ? pages_of(a, b) * blocks_of(b) : 0; };  // of a head, in the line
  const int length0 = length(lane), prefix0 = wave_prefix(length0);
  int64_t total = __builtin_amdgcn_readlane(prefix0, kWave - 1);
  for (int64_t b0 = kWave; b0 < a.batch; b0 += kWave) total += __builtin_amdgcn_readlane(wave_prefix(length(b0 + lane)), kWave - 1);
  total *= heads;
  int64_t share = (total + a.workgroups - 1) / a.workgroups;
  if (share < a.least_share) share = a.least_share;
  int64_t at = blockIdx.x * share, first = 0, b = 0;  // the place in the line; the sequence that holds it, and where that begins
  const int64_t end = at + share < total ? at + share : total;
  if (at < end) {
    int found = 0;
    for (int64_t b0 = 0; found == 0 && b0 < a.batch; b0 += kWave) {
      const int mine = b0 == 0 ? length0 : length(b0 + lane), prefix = b0 == 0 ? prefix0 : wave_prefix(mine);
      const uint64_t holds = __ballot(first + static_cast<int64_t>(prefix) * heads > at);
      if (holds != 0) {
        const int l = __builtin_ctzll(holds);
        found = __builtin_amdgcn_readlane(mine, l);
        b = b0 + l;
        first += static_cast<int64_t>(__builtin_amdgcn_readlane(prefix, l) - found) * heads;
      } else {
        first += static_cast<int64_t>(__builtin_amdgcn_readlane(prefix, kWave - 1)) * heads;
      }
    }
    if (found == 0) return;  // starts or counts changed under the kernel
    int n = pages_of(a, b), blocks = blocks_of(b);
    int block = static_cast<int>((at - first) / n);
    int lo = static_cast<int>((at - first) % n);
    int h = block / blocks;
    block %= blocks;
    while (true) {
      const int64_t left = end - at;
      const int hi = n - lo < left ? n : lo + static_cast<int>(left);
      const int64_t in_sequence = static_cast<int64_t>(h) * a.blocks_of_unit + block, unit = b * heads * a.blocks_of_unit + in_sequence;
      if (lo == 0 && threadIdx.x == 0) a.pieces[unit] = CachePieces{unit + blockIdx.x, (at + n - 1) / share - blockIdx.x + 1};
      f(Piece{b, in_sequence, lo, hi, hi - lo == n, unit + blockIdx.x});
      at += hi - lo;
      if (at >= end) break;
      lo = 0;
      if (++block == blocks) {
        block = 0;
        if (++h == heads) {
          h = 0;
          do {  // the line is not at its end: a sequence with rows and pages follows
            if (++b >= a.batch) return;
            n = pages_of(a, b), blocks = blocks_of(b);
          } while (n == 0 || blocks == 0);
        }
      }
      __syncthreads();
    }
  }
  // blocks that do not stand in the line: no pieces, the join makes zeros of them
  for (b = blockIdx.x; b < a.batch; b += a.workgroups) {
    const int blocks = pages_of(a, b) > 0 ? blocks_of(b) : 0;
    for (int i = threadIdx.x; i < heads * a.blocks_of_unit; i += blockDim.x)
      if (i % a.blocks_of_unit >= blocks) a.pieces[b * heads * a.blocks_of_unit + i] = CachePieces{0, 0};
  }
}

// The lowest n of eight bits, n taken as 0 below 0 and as 8 beyond it.
__device__ __forceinline__ uint32_t low_bits(int n) { return (1u << (n < 0 ? 0 : n > 8 ? 8 : n)) - 1; }

// Which of four bytes are not 0, a bit each.
__device__ __forceinline__ uint32_t true_bytes(uint32_t x) {
  const uint32_t high = (((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u;
  return (high >> 7) * 0x01020408u >> 24 & 15u;  // bits 8 i to 24 + i; no other product of the two reaches bits 24 to 31
}

// Which of kRuns runs of eight keys a row sees, a bit each: run r's stand from first + 16 r on, the row sees those before
// `limit` and, of the drafted ones, those with a true byte in its row of the mask.  A run's bytes are one load, from a
// place so clamped that all eight are the row's.  (With a load for each byte, and the first page's codes loaded after the
// queries, a call of one masked page in 320 tile blocks took 31.0 us instead of 28.6, one of two or three 17.1 instead of 14.6.)
template <int kRuns>
__device__ __forceinline__ uint32_t seen_keys(const CacheAttention& a, const uint8_t* mask_row, int start, int limit, int first) {
  uint32_t seen = 0;
#pragma unroll
  for (int r = 0; r < kRuns; ++r) seen |= low_bits(limit - (first + 16 * r)) << (8 * r);
  if (mask_row == nullptr) return seen;
  uint64_t bytes[kRuns];
  if (a.rows.tokens >= 8) {
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const int at = first + 16 * r - start, from = at < 0 ? 0 : at < a.rows.tokens - 8 ? at : a.rows.tokens - 8;
      __builtin_memcpy(&bytes[r], mask_row + from, 8);
    }
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const int at = first + 16 * r - start, from = at < 0 ? 0 : at < a.rows.tokens - 8 ? at : a.rows.tokens - 8;
      const int up = from - at < 0 ? 0 : from - at > 7 ? 7 : from - at, down = at - from < 0 ? 0 : at - from > 7 ? 7 : at - from;
      bytes[r] = bytes[r] << (8 * up) >> (8 * down);  // by more than seven bytes: none of the run's is the row's
    }
  } else {
    uint64_t row = 0;
#pragma unroll
    for (int i = 0; i < 7; ++i) row |= static_cast<uint64_t>(mask_row[i < a.rows.tokens ? i : a.rows.tokens - 1]) << (8 * i);
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const int at = first + 16 * r - start;
      bytes[r] = row << (8 * (at >= 0 ? 0 : at < -7 ? 7 : -at)) >> (8 * (at <= 0 ? 0 : at > 7 ? 7 : at));
    }
  }
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    const uint32_t drafted = true_bytes(static_cast<uint32_t>(bytes[r])) | true_bytes(static_cast<uint32_t>(bytes[r] >> 32)) << 4;
    seen &= ~((~drafted & 0xffu & ~low_bits(start - (first + 16 * r))) << (8 * r));
  }
  return seen;
}

// A workgroup takes pages of blocks of 16 kTiles rows.  K and V go from memory to the matrix
// instructions' operands in registers: S^T = K Q^T and O^T = V^T P^T, so a lane's scores are already the P that it
// has to give, and the cache's layouts are such that 16 consecutive bytes are a lane's operand.
//   K: lane (m, g) = (lane % 16, lane / 16) takes 16 bytes of row key(m), features 64 c + 16 g on.  Row m of tile t is
//      key 8 (m / 4) + 4 t + m % 4 of the half page: then column n's lane (n, g) holds keys 8 g + 0..7.
//   V: lane (m, g) takes 16 bytes: keys 8 g + 0..7 of features 32 f + 2 m and 32 f + 2 m + 1.
// Bound by the codes' reading: one step at 131072 positions (8 K/V heads of 128) 45.6 us, 6.1 TB/s; 64 steps of up to 8191
// 131.7, 5.3 TB/s.  Plain instead of nontemporal loads read pages at 6.1 instead of 6.8 TB/s.
template <bool kBf16, bool kFp8, int kDim, int kTiles>
struct Stream {
  static constexpr int kChunks = kDim / 64, kFeatures = kDim / 32;  // K pieces of a row; pairs of V tiles
  const CacheAttention& a;
  int n, g;
  uint32_t key_at, value_at, scale_at;  // the lane's first key byte, value byte and scale in half a page
  half8 query[kTiles][kChunks][2];
  float factor[kTiles];            // scores in powers of two: accumulator * key scale * factor
  float top[kTiles], total[kTiles];  // the running maximum; this lane's share of the sum
  float4_t sum[kTiles][2 * kFeatures];
  float reference;  // a power of two no value scale so far is above: sums hold 2^15 / reference times the values
  uint4 key[2][kChunks], value[kFeatures];  // of half a page
  float4 key_scale[2], value_scale[2];

  __device__ __forceinline__ explicit Stream(const CacheAttention& args) : a(args) {
    n = threadIdx.x % 16;
    g = threadIdx.x % kWave / 16;
    key_at = (8 * (n / 4) + n % 4) * kDim + 16 * g;
    value_at = g * (8 * kDim) + 16 * n;
    scale_at = 8 * g;
    reference = 0x1p-100f;
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
      top[r] = kNone;
      total[r] = 0.0f;
#pragma unroll
      for (int f = 0; f < 2 * kFeatures; ++f) sum[r][f] = float4_t{0, 0, 0, 0};
    }
  }

  __device__ __forceinline__ void load_query(int r, const uint16_t* row, bool real) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + 64 * c + 16 * g + 8 * e);
        query[r][c][e] = __builtin_bit_cast(half8, real ? raw : uint4{0, 0, 0, 0});
      }
  }

  __device__ __forceinline__ void scale_query(int r) {
    float largest = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) largest = largest_of<kBf16>(__builtin_bit_cast(uint4, query[r][c][e]), largest);
    const float scale = query_scale(column_max(largest));
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) query[r][c][e] = scaled_halves<kBf16>(__builtin_bit_cast(uint4, query[r][c][e]), scale);
    factor[r] = a.scale * kLog2e / scale;
  }

  __device__ __forceinline__ void load_key(int64_t record, int half) {
    // one address a page in scalar registers, the lane's part of it in 32 bits
    const uint8_t* const k = a.cache.key + record * (kPage * kDim) + 32 * half * kDim;
    const float* const s = a.cache.key_scale + record * kPage + 32 * half;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) key[t][c] = load16(k + (key_at + 4 * t * kDim + 64 * c));
      key_scale[t] = *reinterpret_cast<const float4*>(s + (scale_at + 4 * t));
    }
  }

  __device__ __forceinline__ void load_value(int64_t record, int half) {
    const uint8_t* const v = a.cache.value + record * (kPage * kDim) + 32 * half * kDim;
    const float* const s = a.cache.value_scale + record * kPage + 32 * half;
#pragma unroll
    for (int f = 0; f < kFeatures; ++f) value[f] = load16(v + (value_at + f * 256));
#pragma unroll
    for (int t = 0; t < 2; ++t) value_scale[t] = *reinterpret_cast<const float4*>(s + (scale_at + 4 * t));
  }

  // S^T of the loaded half times the key scales: score[r][t][i] is key 8 g + 4 t + i of row n.
  __device__ __forceinline__ void scores(float4_t (&score)[kTiles][2]) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < kTiles; ++r) score[r][t] = float4_t{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const half8 lo = halves_of<kFp8>(key[t][c].x, key[t][c].y), hi = halves_of<kFp8>(key[t][c].z, key[t][c].w);
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          score[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, query[r][c][0], score[r][t], 0, 0, 0);
          score[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, query[r][c][1], score[r][t], 0, 0, 0);
        }
      }
      const float4 s = key_scale[t];
#pragma unroll
      for (int r = 0; r < kTiles; ++r) score[r][t] *= float4_t{s.x, s.y, s.z, s.w};
    }
  }

  // The softmax's weights of half a page and its share of the sums.  kMasked: bit 4 t + i of seen[r] says whether the row
  // sees key 8 g + 4 t + i; from key `keys` on the half holds nothing that any row sees.
  template <bool kMasked>
  __device__ __forceinline__ void accumulate(float4_t (&score)[kTiles][2], int keys, const uint32_t (&seen)[kTiles]) {
    float scales[2][4], largest = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float s[4] = {value_scale[t].x, value_scale[t].y, value_scale[t].z, value_scale[t].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        scales[t][i] = kMasked && 8 * g + 4 * t + i >= keys ? 0.0f : s[i];
        largest = fmaxf(largest, scales[t][i]);
      }
    }
    largest = column_max(largest);
    const float above = __uint_as_float((__float_as_uint(largest) & 0x7f800000u) + 0x00800000u);
    const float next_reference = fmaxf(reference, above);
    const float inverse = __builtin_amdgcn_rcpf(next_reference);  // exact: a power of two
    const float shrink = reference * inverse;
    bool changed = next_reference > reference;
    reference = next_reference;
    const float unit = 0x1p15f * inverse;

    half8 weight[kTiles];
    float keep[kTiles];
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
      float page_top = kNone;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kMasked)
            if ((seen[r] >> (4 * t + i) & 1) == 0) score[r][t][i] = kNone;
          page_top = fmaxf(page_top, score[r][t][i]);
        }
      const float next = fmaxf(top[r], column_max(page_top) * factor[r]);
      const float base = next == kNone ? 0.0f : next;
      keep[r] = exp2_fast(top[r] - base);
      changed = changed || next > top[r];
      top[r] = next;
      total[r] *= keep[r];
      keep[r] *= shrink;
      uint32_t packed[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float s = score[r][t][i];
          // an unseen key's score is -inf, also times the factor; its value scale may be anything
          const float p = exp2_fast(fmaf(s, factor[r], -base));
          total[r] += p;
          w[i] = p * (scales[t][i] * unit);
          if constexpr (kMasked) w[i] = s == kNone ? 0.0f : w[i];
        }
        packed[2 * t] = pack_half2(w[0], w[1]);
        packed[2 * t + 1] = pack_half2(w[2], w[3]);
      }
      weight[r] = __builtin_bit_cast(half8, uint4{packed[0], packed[1], packed[2], packed[3]});
    }
    if (__any(changed)) {
#pragma unroll
      for (int r = 0; r < kTiles; ++r)
#pragma unroll
        for (int f = 0; f < 2 * kFeatures; ++f) sum[r][f] *= keep[r];
    }
    // codes of slots that hold nothing could be FP8 NaN, which zero weights do not cancel
    const int held = keys - 8 * g;
    const uint32_t low = held >= 4 ? ~0u : held <= 0 ? 0u : (1u << (8 * held)) - 1;
    const uint32_t high = held >= 8 ? ~0u : held <= 4 ? 0u : (1u << (8 * (held - 4))) - 1;
#pragma unroll
    for (int f = 0; f < kFeatures; ++f) {
      uint4 v = value[f];
      if constexpr (kMasked && kFp8) v = uint4{v.x & low, v.y & high, v.z & low, v.w & high};
      const half8 even = halves_of<kFp8>(v.x, v.y), odd = halves_of<kFp8>(v.z, v.w);
#pragma unroll
      for (int r = 0; r < kTiles; ++r) {
        sum[r][2 * f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, weight[r], sum[r][2 * f], 0, 0, 0);
        sum[r][2 * f + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, weight[r], sum[r][2 * f + 1], 0, 0, 0);
      }
    }
  }
};

template <int kDim>
struct Shared {  // a row tile's sums of each wave
  float sum[kWaves][16][kDim + 4];
  float top[kWaves][16], total[kWaves][16];
};

template <bool kBf16, bool kFp8, int kDim, int kTiles, bool kSelected>
__device__ __forceinline__ void cache_stream_block(const CacheAttention& a, const Piece& piece, Shared<kDim>& shared) {
  constexpr int kRows = 16 * kTiles;
  const int wave = threadIdx.x / kWave;
  const int group = a.heads / a.cache.kv_heads;
  const int unit_rows = (kSelected ? 1 : a.rows.tokens) * group;
  const int first_row = static_cast<int>(piece.block % a.blocks_of_unit) * kRows;
  const int64_t b = piece.b, unit = piece.block / a.blocks_of_unit;  // of the sequence
  const int first_token = kSelected ? static_cast<int>(unit % a.rows.tokens) : 0;
  const int64_t h = kSelected ? unit / a.rows.tokens : unit;
  int hi = piece.hi;

  // page numbers of the wave's first three steps, before anything waits for where the rows stand
  const int32_t* const selected = a.selected + (b * a.cache.kv_heads * a.rows.tokens + unit) * a.budget;
  const int32_t* const table = a.rows.page_table + b * a.rows.table_stride;
  const auto name = [&](int step) {
    if constexpr (!kSelected) return step;
    return selected[step < a.budget ? step : a.budget - 1];
  };
  const auto entry = [&](int logical) { return table[logical < 0 ? 0 : logical < a.rows.table_width ? logical : a.rows.table_width - 1]; };
  const auto record = [&](int page) { return (page >= 0 && page < a.rows.pages ? page : 0) * static_cast<int64_t>(a.cache.kv_heads) + h; };
  const int first_step = piece.lo + __builtin_amdgcn_readfirstlane(wave);
  int step = first_step;
  const int logical0 = name(step);
  int logical1 = name(step + kWaves), logical2 = name(step + 2 * kWaves);
  int page = entry(logical0), page1 = entry(logical1);

  Stream<kBf16, kFp8, kDim, kTiles> s(a);
  const int start = a.rows.starts[b];
  const int count = a.rows.count(b);
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    const int row = first_row + 16 * r + s.n;
    const uint16_t* q = static_cast<const uint16_t*>(a.query.data) + b * a.query.stride_batch;
    if (row < unit_rows) q += (h * group + row % group) * a.query.stride_head + (first_token + row / group) * a.query.stride_seq;  // else any row, as zeros
    s.load_query(r, q, row < unit_rows);
  }
  if (step < hi) {
    s.load_key(record(page), 0);
    s.load_value(record(page), 0);
  }
  int most = 0, least = 0;  // the largest limit, and what every row with a limit sees stands before
  {
    const int last = first_row + kRows < unit_rows ? first_row + kRows - 1 : unit_rows - 1;
    const int first_t = first_token + first_row / group;
    const int last_t = first_token + last / group < count ? first_token + last / group : count - 1;
    if (first_t < count) {
      most = static_cast<int>(a.rows.end(b, a.mask != nullptr ? count - 1 : last_t));
      least = a.mask != nullptr ? (start < most ? (start > 0 ? start : 0) : most) : static_cast<int>(a.rows.end(b, first_t));
    }
  }
  const int end_page = (most + kPage - 1) / kPage, whole_pages = least / kPage;
  if (!kSelected && hi > end_page) hi = end_page;

  // First the pages of which every row sees every key, in a stream: a wave's pages come step by step, the codes half a
  // page before they are used and the page's number two steps before that.  Every load of the loop is made in every
  // step, where there is no page from a clamped place (the list's last entry, page 0): a load on a branch would make
  // each wait a wait for all loads.
  const auto is_page = [&](int logical, int page) { return logical >= 0 && logical < end_page && page >= 0 && page < a.rows.pages; };
  const int stop = kSelected || hi < whole_pages ? hi : whole_pages;
  {
    bool here = step < stop && logical0 < whole_pages && is_page(logical0, page);
#pragma unroll
    for (int r = 0; r < kTiles; ++r) s.scale_query(r);
    const uint32_t none[kTiles] = {};
    for (; step < stop; step += kWaves) {
      const int page2 = entry(logical2), logical3 = name(step + 3 * kWaves);
      const bool next = step + kWaves < stop && logical1 < whole_pages && is_page(logical1, page1);
      const int64_t now = record(page), after = record(page1);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float4_t score[kTiles][2];
        if (here) s.scores(score);
        s.load_key(half == 0 ? now : after, 1 - half);
        if (here) s.template accumulate<false>(score, 32, none);
        s.load_value(half == 0 ? now : after, 1 - half);
      }
      logical1 = logical2;
      logical2 = logical3;
      page = page1;
      page1 = page2;
      here = next;
    }
  }
  // then those of which some row sees a part: of a range the last ones, of a list any
  if (kSelected) step = first_step;
  int limit[kTiles];  // what the lane's row of each tile sees stands before this position
  const uint8_t* mask_row[kTiles];
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    const int row = first_row + 16 * r + s.n, token = first_token + row / group;
    const bool real = row < unit_rows && token < count;
    limit[r] = real ? static_cast<int>(a.rows.end(b, a.mask != nullptr ? count - 1 : token)) : 0;
    mask_row[r] = a.mask != nullptr ? a.mask + b * a.mask_stride_batch + (real ? token * a.mask_stride_row : 0) : nullptr;
  }
  for (; step < hi; step += kWaves) {
    const int logical = name(step), page = entry(logical);
    if (!is_page(logical, page) || logical < whole_pages) continue;
    for (int half = 0; half < 2; ++half) {
      const int base = logical * kPage + 32 * half;
      const int keys = most - base < 32 ? most - base : 32;
      if (keys <= 0) break;
      s.load_key(record(page), half);
      s.load_value(record(page), half);
      uint32_t seen[kTiles];
#pragma unroll
      for (int r = 0; r < kTiles; ++r) seen[r] = seen_keys<1>(a, mask_row[r], start, limit[r], base + 8 * s.g);
      float4_t score[kTiles][2];
      s.scores(score);
      s.template accumulate<true>(score, keys, seen);
    }
  }

  // the waves' sums joined, a row tile at a time: 16 threads a row
  constexpr int kPer = kDim / 16;
  const int row16 = threadIdx.x / 16, piece16 = threadIdx.x % 16;
#pragma unroll
  for (int r = 0; r < kTiles; ++r) {
    const float total = column_sum(s.total[r]);
    const float value_unit = s.reference * 0x1p-15f;
    if (r > 0) __syncthreads();
    if (s.g == 0) {
      shared.top[wave][s.n] = s.top[r];
      shared.total[wave][s.n] = total;
    }
#pragma unroll
    for (int f = 0; f < kDim / 32; ++f) {
      const float4_t even = s.sum[r][2 * f], odd = s.sum[r][2 * f + 1];
      float4* const to = reinterpret_cast<float4*>(&shared.sum[wave][s.n][32 * f + 8 * s.g]);
      to[0] = float4{even[0] * value_unit, odd[0] * value_unit, even[1] * value_unit, odd[1] * value_unit};
      to[1] = float4{even[2] * value_unit, odd[2] * value_unit, even[3] * value_unit, odd[3] * value_unit};
    }
    __syncthreads();
    const int row = first_row + 16 * r + row16;
    if (row >= unit_rows) continue;
    float top = kNone;
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, shared.top[w][row16]);
    const float base = top == kNone ? 0.0f : top;
    float joined = 0.0f, x[kPer] = {};
    for (int w = 0; w < kWaves; ++w) {
      const float scale = exp2_fast(shared.top[w][row16] - base);
      joined += shared.total[w][row16] * scale;
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = fmaf(shared.sum[w][row16][piece16 * kPer + e], scale, x[e]);
    }
    const int t = first_token + row / group;
    if (!piece.whole) {
      const int64_t to_row = piece.index * kRows + 16 * r + row16;
      float* const to = a.partial + to_row * kDim + piece16 * kPer;
#pragma unroll
      for (int e = 0; e < kPer; e += 4) *reinterpret_cast<float4*>(to + e) = float4{x[e], x[e + 1], x[e + 2], x[e + 3]};
      if (piece16 == 0) a.partial_stats[to_row] = float2{top, joined};
      continue;
    }
    // a row beyond the count has gone through the pages that every real row sees, whatever they hold
    const bool none = joined == 0.0f || t >= count;
    const float inverse = 1.0f / joined;
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = none ? 0.0f : x[e] * inverse;
    uint16_t* const out = static_cast<uint16_t*>(a.output) + ((b * a.heads + h * group + row % group) * a.rows.tokens + t) * kDim + piece16 * kPer;
#pragma unroll
    for (int e = 0; e < kPer; e += 4)
      *reinterpret_cast<uint2*>(out + e) = uint2{narrow2<kBf16>(x[e], x[e + 1]), narrow2<kBf16>(x[e + 2], x[e + 3])};
  }
}

// ---- many rows --------------------------------------------------------------------------------------------------------
//
// Blocks of 128 or 256 rows: each of a workgroup's four or eight waves has 32 and goes through all of its pages.  A
// page's codes are widened once, by all waves, into halves in LDS, two pages in turn: while one is used, the next one's
// codes, loaded a page earlier, are widened into the other, and the ones after that are loaded.  S^T = K Q^T and
// O^T = V^T P^T on 32x32x16 instructions; lane (n, g) = (lane % 32, lane / 32) holds of row n the keys 16 p + 8 g + 0..7
// of each 32.
// Bound by VALU issue (widening, softmax, P: 55 - 69% of the time) beside the matrix instructions (33 - 36%), which hide only part of
// it: 2048 rows of 32 heads on 8 of 128 after 32768 positions 1266 us, 896 TFLOP/s, 1.33 ms with each read just before its
// matrix instruction.  Waves in opposite halves of a page took 1.31 - 1.50 ms, 16 rows a wave at four waves a SIMD 1.76.

typedef float float16_t __attribute__((ext_vector_type(16)));

template <int kDim>
struct TileShared {
  half8 key[2][kPage][kDim / 8];    // row m of the matrix instructions: key m with bits 2 and 3 exchanged; 16-byte pieces
                                    // exchanged within eight by the row, so that eight rows' same piece is in all banks
  half8 value[2][kPage / 8][kDim];  // eight keys of a feature
  float key_scale[2][kPage], value_scale[2][kPage];  // the values' in units of 2^-15 of the reference
};

// The order of a block of kReads LDS reads that feed as many matrix instructions: six reads ahead, or the scheduler, to
// save registers, waits for each pair's.
template <int kReads>
__device__ __forceinline__ void reads_ahead() {
  constexpr int kDsRead = 0x100, kMatrix = 0x8, kAhead = 6;
  __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
  for (int i = kAhead; i < kReads; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMatrix, kAhead, 0);
}

template <bool kBf16, bool kFp8, int kDim, int kTileWaves>
struct Tile {
  static constexpr int kSteps = kDim / 16, kFeatures = kDim / 32;
  static constexpr int kEights = kPage * kDim / 8 / (kWave * kTileWaves);  // a thread's share of a page: this many 8 codes
  const CacheAttention& a;
  TileShared<kDim>& shared;
  int n, g;
  half8 query[kSteps];
  float factor, top, total;
  float reference, sum_reference;  // see Stream: of the page widened last, and what the sums are in
  float16_t sum[kFeatures];
  uint2 key[kEights], value[kEights];  // codes of the page to come
  float key_scale, value_scale;

  __device__ __forceinline__ Tile(const CacheAttention& args, TileShared<kDim>& lds) : a(args), shared(lds) {
    n = threadIdx.x % 32;
    g = threadIdx.x % kWave / 32;
    top = kNone;
    total = 0.0f;
    reference = sum_reference = 0x1p-100f;
#pragma unroll
    for (int f = 0; f < kFeatures; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[f][i] = 0.0f;
  }

  __device__ __forceinline__ void load_query(const uint16_t* row, bool real) {
    uint4 raw[kSteps];
    float largest = 0.0f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) raw[k] = *reinterpret_cast<const uint4*>(row + 16 * k + 8 * g);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) largest = largest_of<kBf16>(raw[k], largest);
    const float scale = query_scale(cross_half_max(real ? largest : 0.0f));
#pragma unroll
    for (int k = 0; k < kSteps; ++k) query[k] = scaled_halves<kBf16>(real ? raw[k] : uint4{0, 0, 0, 0}, scale);
    factor = a.scale * kLog2e / scale;
  }

  __device__ __forceinline__ void load(int64_t record) {
    const uint8_t* const k = a.cache.key + record * (kPage * kDim);
    const uint8_t* const v = a.cache.value + record * (kPage * kDim);
    if constexpr (kEights == 1) {
      key[0] = *reinterpret_cast<const uint2*>(k + threadIdx.x * 8);
      value[0] = *reinterpret_cast<const uint2*>(v + threadIdx.x * 8);
    } else {
#pragma unroll
      for (int i = 0; i < kEights; i += 2) {
        const uint4 x = *reinterpret_cast<const uint4*>(k + (threadIdx.x * (8 * kEights) + 8 * i));
        const uint4 y = *reinterpret_cast<const uint4*>(v + (threadIdx.x * (8 * kEights) + 8 * i));
        key[i] = uint2{x.x, x.y};
        key[i + 1] = uint2{x.z, x.w};
        value[i] = uint2{y.x, y.y};
        value[i + 1] = uint2{y.z, y.w};
      }
    }
    key_scale = (a.cache.key_scale + record * kPage)[threadIdx.x % kPage];
    value_scale = (a.cache.value_scale + record * kPage)[threadIdx.x % kPage];
  }

  // Slots from `keys` on hold nothing that any row sees; their codes could be FP8 NaN.
  __device__ __forceinline__ void widen(int buffer, int keys) {
#pragma unroll
    for (int i = 0; i < kEights; ++i) {
      const int at = threadIdx.x * kEights + i, slot = at / (kDim / 8), piece = at % (kDim / 8);
      const int row = (slot & ~12) | (slot & 4) << 1 | (slot & 8) >> 1;
      shared.key[buffer][row][piece ^ (row & 7)] = halves_of<kFp8>(key[i].x, key[i].y);
      uint2 v = value[i];
      if constexpr (kFp8) {
        const int held = keys - 8 * (at / kDim);
        v.x &= held >= 4 ? ~0u : held <= 0 ? 0u : (1u << (8 * held)) - 1;
        v.y &= held >= 8 ? ~0u : held <= 4 ? 0u : (1u << (8 * (held - 4))) - 1;
      }
      shared.value[buffer][at / kDim][at % kDim] = halves_of<kFp8>(v.x, v.y);
    }
    // every wave has all 64 value scales
    const float held = static_cast<int>(threadIdx.x % kPage) >= keys ? 0.0f : value_scale;
    const float largest = wave_max(held);
    const float above = __uint_as_float((__float_as_uint(largest) & 0x7f800000u) + 0x00800000u);
    reference = fmaxf(reference, above);
    if (threadIdx.x < kPage) {
      shared.key_scale[buffer][threadIdx.x] = key_scale;
      shared.value_scale[buffer][threadIdx.x] = held * (0x1p15f * __builtin_amdgcn_rcpf(reference));  // exact: a power of two
    }
  }

  // A page in LDS: score[kt][8 p + j] is key 32 kt + 16 p + 8 g + j of row n.  `unit`: its reference.
  // kMasked: bit 16 kt + 8 p + j of `seen` says whether the row sees it.
  template <bool kMasked>
  __device__ __forceinline__ void use(int buffer, float unit, uint32_t seen) {
    float16_t score[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) score[kt][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        score[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(shared.key[buffer][32 * kt + n][(2 * k + g) ^ (n & 7)], query[k], score[kt], 0, 0, 0);
    reads_ahead<2 * kSteps>();
    // eight keys' scales stand together; read ahead of their use, which the scheduler would put off to save registers
    float4 scales[2][2][2];
    const auto read = [&](const float (&from)[kPage]) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int q = 0; q < 2; ++q) scales[kt][p][q] = *reinterpret_cast<const float4*>(&from[32 * kt + 16 * p + 8 * g + 4 * q]);
      __builtin_amdgcn_sched_barrier(0);
    };
    read(shared.key_scale[buffer]);
    float page_top = kNone;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 s = scales[kt][p][q];
          const float ks[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 8 * p + 4 * q + i;
            float x = score[kt][at] * ks[i];
            if constexpr (kMasked) x = seen >> (16 * kt + at) & 1 ? x : kNone;
            score[kt][at] = x;
            page_top = fmaxf(page_top, x);
          }
        }
    read(shared.value_scale[buffer]);
    const float next = fmaxf(top, cross_half_max(page_top) * factor);
    const float base = next == kNone ? 0.0f : next;
    const float keep = exp2_fast(top - base);
    if (__any(next > top || unit > sum_reference)) {
      const float scale = keep * (sum_reference * __builtin_amdgcn_rcpf(unit));
#pragma unroll
      for (int f = 0; f < kFeatures; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[f][i] *= scale;
      total *= keep;
    }
    top = next;
    sum_reference = unit;
    half8 weight[2][2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t packed[4];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 s = scales[kt][p][q];
          const float vs[4] = {s.x, s.y, s.z, s.w};
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = score[kt][8 * p + 4 * q + i];
            const float e = exp2_fast(fmaf(x, factor, -base));
            total += e;
            w[i] = e * vs[i];
            if constexpr (kMasked) w[i] = x == kNone ? 0.0f : w[i];
          }
          packed[2 * q] = pack_half2(w[0], w[1]);
          packed[2 * q + 1] = pack_half2(w[2], w[3]);
        }
        weight[kt][p] = __builtin_bit_cast(half8, uint4{packed[0], packed[1], packed[2], packed[3]});
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int f = 0; f < kFeatures; ++f)
          sum[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(shared.value[buffer][4 * kt + 2 * p + g][32 * f + n], weight[kt][p], sum[f], 0, 0, 0);
    reads_ahead<4 * kFeatures>();
  }
};

template <bool kBf16, bool kFp8, int kDim, int kTileWaves>
__device__ __forceinline__ void cache_tile_block(const CacheAttention& a, const Piece& piece, TileShared<kDim>& shared) {
  constexpr int kTileRows = 32 * kTileWaves;
  const int group = a.heads / a.cache.kv_heads;
  const int unit_rows = a.rows.tokens * group;
  const int first_row = static_cast<int>(piece.block % a.blocks_of_unit) * kTileRows;
  const int64_t b = piece.b, h = piece.block / a.blocks_of_unit;
  const int start = a.rows.starts[b], count = a.rows.count(b);
  Tile<kBf16, kFp8, kDim, kTileWaves> s(a, shared);
  // Two pages in turn; a place past the last is loaded from a clamped one, and a page that the table does not name from
  // page 0 and not used.  The first is on its way before anything waits for the rows.
  const int32_t* const table = a.rows.page_table + b * a.rows.table_stride;
  const auto entry = [&](int logical) { return table[logical < a.rows.table_width ? logical : a.rows.table_width - 1]; };
  const auto is_page = [&](int page) { return page >= 0 && page < a.rows.pages; };
  const auto record = [&](int page) { return (is_page(page) ? page : 0) * static_cast<int64_t>(a.cache.kv_heads) + h; };
  int step = piece.lo;
  int page = entry(step), page1 = entry(step + 1), page2 = entry(step + 2);
  s.load(record(page));
  const int row = first_row + 32 * (threadIdx.x / kWave) + s.n;
  const int token = row / group;
  const bool real = row < unit_rows && token < count;
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.query.data) + b * a.query.stride_batch;
    if (row < unit_rows) q += (h * group + row % group) * a.query.stride_head + token * a.query.stride_seq;  // else any row, as zeros
    s.load_query(q, row < unit_rows);
  }
  int most = 0, least = 0;  // as in cache_stream_block
  {
    const int last = first_row + kTileRows < unit_rows ? first_row + kTileRows - 1 : unit_rows - 1;
    const int first_t = first_row / group, last_t = last / group < count ? last / group : count - 1;
    if (first_t < count) {
      most = static_cast<int>(a.rows.end(b, a.mask != nullptr ? count - 1 : last_t));
      least = a.mask != nullptr ? (start < most ? (start > 0 ? start : 0) : most) : static_cast<int>(a.rows.end(b, first_t));
    }
  }
  const int end_page = (most + kPage - 1) / kPage, whole_pages = least / kPage;
  const int hi = piece.hi < end_page ? piece.hi : end_page;
  const bool busy = __ballot(real) != 0;  // a wave without rows keeps the others' pace

  if (piece.lo < hi) {
    s.widen(step & 1, most - step * kPage);
    s.load(record(page1));
    __syncthreads();
    const auto then = [&] {  // the pages after this one, a step further
      const int page3 = entry(step + 3);
      s.widen(~step & 1, most - (step + 1) * kPage);
      s.load(record(page2));
      page = page1;
      page1 = page2;
      page2 = page3;
      __syncthreads();
    };
    for (; step < hi && step < whole_pages; ++step) {
      if (is_page(page) && busy) s.template use<false>(step & 1, s.reference, 0);
      then();
    }
    const uint8_t* const mask_row =
        a.mask != nullptr ? a.mask + b * a.mask_stride_batch + (real ? token * a.mask_stride_row : 0) : nullptr;
    const int limit = real ? static_cast<int>(a.rows.end(b, a.mask != nullptr ? count - 1 : token)) : 0;
    for (; step < hi; ++step) {  // some row sees a part
      if (is_page(page) && busy) {
        const uint32_t seen = seen_keys<4>(a, mask_row, start, limit, step * kPage + 8 * s.g);
        __builtin_amdgcn_sched_barrier(0);  // its 32 bytes are one register before the scores are more
        s.template use<true>(step & 1, s.reference, seen);
      }
      then();
    }
  }

  const float total = cross_half_sum(s.total);
  if (row >= unit_rows) return;
  if (!piece.whole) {
    const float value_unit = s.sum_reference * 0x1p-15f;
    const int64_t to_row = piece.index * kTileRows + row - first_row;
    float* const to = a.partial + to_row * kDim + 4 * s.g;
#pragma unroll
    for (int f = 0; f < kDim / 32; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(to + 32 * f + 8 * i) = float4{s.sum[f][4 * i] * value_unit, s.sum[f][4 * i + 1] * value_unit,
                                                                 s.sum[f][4 * i + 2] * value_unit, s.sum[f][4 * i + 3] * value_unit};
    if (s.g == 0) a.partial_stats[to_row] = float2{s.top, total};
    return;
  }
  // a row beyond the count has gone through the pages that every real row sees, whatever they hold
  const bool none = total == 0.0f || !real;
  const float inverse = s.sum_reference * 0x1p-15f / total;
  uint16_t* const out = static_cast<uint16_t*>(a.output) + ((b * a.heads + h * group + row % group) * a.rows.tokens + token) * kDim + 4 * s.g;
#pragma unroll
  for (int f = 0; f < kDim / 32; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = none ? 0.0f : s.sum[f][4 * i + e] * inverse;
      *reinterpret_cast<uint2*>(out + 32 * f + 8 * i) = uint2{narrow2<kBf16>(x[0], x[1]), narrow2<kBf16>(x[2], x[3])};
    }
}

// ---- kernels ----------------------------------------------------------------------------------------------------------

enum class Pages { kAll, kLine, kList };  // every page, or a line's share of them; pages from a list

// Hands a workgroup its pieces.
template <Pages kPages, typename F>
__device__ __forceinline__ void share_out(const CacheAttention& a, int block_rows, F f) {
  constexpr bool kList = kPages == Pages::kList;
  if constexpr (kPages == Pages::kLine) {
    walk_line(a, block_rows, f);
    return;
  }
  const int64_t blocks = static_cast<int64_t>(a.cache.kv_heads) * a.blocks_of_unit * (kList ? a.rows.tokens : 1);  // of a sequence
  const int64_t unit = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t b = unit / blocks;
  const int n = kList ? listed_pages(a, unit) : pages_of(a, b);
  int parts = (n + a.least_share - 1) / a.least_share;
  parts = parts < 1 ? 1 : parts < a.parts ? parts : a.parts;
  if (part == 0 && threadIdx.x == 0 && a.shares != CacheShares::kWhole) a.pieces[unit] = CachePieces{unit * a.parts, parts};
  if (part >= parts) return;
  const int lo = static_cast<int>(static_cast<int64_t>(n) * part / parts), hi = static_cast<int>(static_cast<int64_t>(n) * (part + 1) / parts);
  f(Piece{b, unit % blocks, lo, hi, parts == 1, unit * a.parts + part});
}

template <bool kBf16, bool kFp8, int kDim, int kTiles, Pages kPages>
__global__ __launch_bounds__(kWave* kWaves, kTiles == 1 && kPages != Pages::kLine ? 3 : 2) void cache_stream_kernel(CacheAttention a) {
  __shared__ Shared<kDim> shared;
  share_out<kPages>(a, 16 * kTiles, [&](const Piece& piece) { cache_stream_block<kBf16, kFp8, kDim, kTiles, kPages == Pages::kList>(a, piece, shared); });
}

template <bool kBf16, bool kFp8, int kDim, int kTileWaves, Pages kPages>
__global__ __launch_bounds__(kWave* kTileWaves, 2) void cache_tile_kernel(CacheAttention a) {
  __shared__ TileShared<kDim> shared;
  share_out<kPages>(a, 32 * kTileWaves, [&](const Piece& piece) { cache_tile_block<kBf16, kFp8, kDim, kTileWaves>(a, piece, shared); });
}

// The pieces of split blocks joined: kJoin waves per row, each every kJoin-th piece.
template <bool kBf16, int kDim, bool kSelected, int kJoin>
__global__ __launch_bounds__(kWave* kWaves) void cache_join_kernel(CacheAttention a, int block_rows) {
  constexpr int kPer = kDim / kWave;
  __shared__ float shared_sum[kWaves][kDim], shared_total[kWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int group = a.heads / a.cache.kv_heads;
  const int64_t row_of_call = static_cast<int64_t>(blockIdx.x) * (kWaves / kJoin) + (kJoin == 1 ? wave : 0);
  if (row_of_call >= static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens) return;
  const int64_t pair = row_of_call / (static_cast<int64_t>(a.rows.tokens) * group), b = pair / a.cache.kv_heads, h = pair % a.cache.kv_heads;
  const int within = static_cast<int>(row_of_call % (static_cast<int64_t>(a.rows.tokens) * group)), t = within / group;
  const int row = kSelected ? within % group : within;
  const int64_t unit = kSelected ? pair * a.rows.tokens + t : pair;
  const CachePieces pieces = a.pieces[unit * a.blocks_of_unit + row / block_rows];
  if (pieces.parts == 1) return;
  const int parts = t < a.rows.count(b) ? pieces.parts : 0;  // 0 pieces: a sequence without pages
  const int64_t first_row = pieces.first * block_rows + row % block_rows;
  float top = kNone;
  for (int p = lane; p < parts; p += kWave) top = fmaxf(top, a.partial_stats[first_row + static_cast<int64_t>(p) * block_rows].x);
  top = wave_max(top);
  const float base = top == kNone ? 0.0f : top;
  float total = 0.0f, x[kPer] = {};
#pragma unroll 4
  for (int p = kJoin == 1 ? 0 : wave; p < parts; p += kJoin) {
    const int64_t at = first_row + static_cast<int64_t>(p) * block_rows;
    const float2 stats = a.partial_stats[at];
    const float scale = exp2_fast(stats.x - base);
    total = fmaf(stats.y, scale, total);
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = fmaf(a.partial[at * kDim + lane * kPer + e], scale, x[e]);
  }
  uint16_t* const out = static_cast<uint16_t*>(a.output) + ((b * a.heads + h * group + within % group) * a.rows.tokens + t) * kDim;
  if constexpr (kJoin == 1) {
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    const uint32_t packed = narrow2<kBf16>(total == 0.0f ? 0.0f : x[0] * inverse, total == 0.0f ? 0.0f : x[kPer - 1] * inverse);
    if constexpr (kPer == 2)
      reinterpret_cast<uint32_t*>(out)[lane] = packed;
    else
      out[lane] = static_cast<uint16_t>(packed);
    return;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) shared_sum[wave][lane * kPer + e] = x[e];
  if (lane == 0) shared_total[wave] = total;
  __syncthreads();
  if (threadIdx.x >= kDim / 2) return;
  total = 0.0f;
  float low = 0.0f, high = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    total += shared_total[w];
    low += shared_sum[w][2 * threadIdx.x];
    high += shared_sum[w][2 * threadIdx.x + 1];
  }
  const float inverse = 1.0f / total;
  reinterpret_cast<uint32_t*>(out)[threadIdx.x] = total == 0.0f ? 0u : narrow2<kBf16>(low * inverse, high * inverse);
}

}  // namespace

// Rows of a unit.
static int64_t unit_rows(const CacheAttention& a) {
  return (a.selected != nullptr ? 1 : static_cast<int64_t>(a.rows.tokens)) * (a.heads / a.cache.kv_heads);
}

// Rows of a block: the stream kernel's 16 or 32 (up to two blocks of them: the second reads its codes from the caches),
// or the tile kernel's 128 or 256.  Measured at 8 K/V heads of 128 (us):
//   rows  sequences  context   32 a block  128 a block
//     48          8     8192         54.5         70.5
//     64          8     8192         57           72
//     64          1    16384         24.4         41.5
//     64         64     4096        180          177
//     96          8     8192         72 - 75.6    74.6    (three blocks of 32)
// and with 256 rows, which 128-row blocks read twice: full sequences, 64 of 4096, 454 for 128 and 398 for 256; ragged ones 276
// and 320; 8 of 8192 143 and 130; one of 16384 65 and 59.
static int block_rows(const CacheAttention& a) {
  const int64_t rows = unit_rows(a);
  return rows <= 16 ? 16 : rows <= 64 || a.selected != nullptr ? 32 : rows <= 128 ? 128 : 256;
}

// Up to kUnsplit pages stay one workgroup's: split, they cost the join's launch (4 us; 5 pages in one workgroup 6.6 us, in
// two and joined 9.4).  Beyond that parts go down to kLeastShare pages, one for each wave: at least 16 a part took 24
// instead of 14.5 us for 14 blocks of 17 pages, 29 instead of 19.4 for 26 of up to 29.
//
// One sequence's blocks, and lists of selected pages, are of a length: equal parts, as many workgroups as a CU takes
// one of (two of 128 rows).  Two and three a CU took 54.1 and 57.8 instead of 51.8 us for a step of 131072 positions, 35.2 and 37.0
// instead of 34.8 for selected pages: there are more parts to join.  Sequences of different lengths share a line: one, two and three
// workgroups a CU took 153, 134 - 139 and 134 - 156 us for 64 steps of up to 8192 positions.  Where there are eight
// blocks to a place and more, the places fill without splitting.
constexpr int kUnsplit = 16, kLeastShare = 4;

CacheParts cache_attention_parts(const CacheAttention& a, int head_dim, int cus) {
  const int rows = block_rows(a);
  const int64_t units = static_cast<int64_t>(a.batch) * a.cache.kv_heads * (a.selected != nullptr ? a.rows.tokens : 1);
  CacheParts p{};
  p.blocks_of_unit = ceil_div(unit_rows(a), rows);
  const int64_t blocks = units * p.blocks_of_unit, pages = a.selected != nullptr ? a.budget : a.rows.table_width;
  p.least_share = kLeastShare;
  p.shares = CacheShares::kWhole;
  p.parts = 1;
  p.workgroups = blocks;
  if (pages <= kUnsplit) return p;
  if (a.batch == 1 || a.selected != nullptr) {
    const int64_t slots = static_cast<int64_t>(cus) * (rows == 128 ? 2 : 1);
    p.parts = std::min(slots / blocks, ceil_div(pages, p.least_share));
    if (p.parts <= 1) {
      p.parts = 1;
      return p;
    }
    p.shares = CacheShares::kEven;
    p.workgroups = blocks * p.parts;
    p.rows = p.workgroups * rows;
  } else {
    const int64_t slots = static_cast<int64_t>(cus) * (rows == 256 ? 1 : 2);
    if (blocks >= 8 * slots) return p;
    if (pages * p.blocks_of_unit > INT32_MAX / kWave) return p;  // walk_line adds a wave's lengths in 32 bits
    p.shares = CacheShares::kLine;
    p.workgroups = std::min(slots, ceil_div(blocks * pages, p.least_share));
    p.rows = (blocks + p.workgroups) * rows;
  }
  p.bytes = p.rows * (head_dim + 2) * 4 + blocks * sizeof(CachePieces);
  return p;
}

hipError_t launch_cache_attention(const CacheAttention& a, CacheForm form, hipStream_t stream) {
  const dim3 blocks(static_cast<uint32_t>(a.workgroups)), threads(kWave * kWaves);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens;
  const int of_block = block_rows(a);
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    constexpr bool kBf16 = decltype(bf16)::value, kFp8 = decltype(fp8)::value;
    constexpr int kDim = decltype(dim)::value;
    const auto run = [&](auto pages) {
      constexpr Pages kPages = decltype(pages)::value;
      constexpr bool kList = kPages == Pages::kList;
      if (of_block == 16)
        cache_stream_kernel<kBf16, kFp8, kDim, 1, kPages><<<blocks, threads, 0, stream>>>(a);
      else if (of_block == 32)
        cache_stream_kernel<kBf16, kFp8, kDim, 2, kPages><<<blocks, threads, 0, stream>>>(a);
      else if constexpr (!kList) {
        if (of_block == 128)
          cache_tile_kernel<kBf16, kFp8, kDim, 4, kPages><<<blocks, dim3(256), 0, stream>>>(a);
        else
          cache_tile_kernel<kBf16, kFp8, kDim, 8, kPages><<<blocks, dim3(512), 0, stream>>>(a);
      }
      if (const hipError_t err = hipGetLastError(); err != hipSuccess || a.shares == CacheShares::kWhole) return err;
      if (a.parts > 4)  // a workgroup a row: else a wave goes through all the parts of one
        cache_join_kernel<kBf16, kDim, kList, kWaves><<<dim3(static_cast<uint32_t>(rows)), threads, 0, stream>>>(a, of_block);
      else
        cache_join_kernel<kBf16, kDim, kList, 1><<<dim3(static_cast<uint32_t>(ceil_div(rows, kWaves))), threads, 0, stream>>>(a, of_block);
      return hipGetLastError();
    };
    if (a.selected != nullptr) return run(std::integral_constant<Pages, Pages::kList>{});
    if (a.shares == CacheShares::kLine) return run(std::integral_constant<Pages, Pages::kLine>{});
    return run(std::integral_constant<Pages, Pages::kAll>{});
  });
}

}  // namespace piper
