// Device helpers of the quantised cache and the launchers its C entry points call.
#pragma once

#include "cache.h"
#include "kernels.h"
#include "quant.h"

namespace piper {

struct Cache {
  uint8_t* key;
  float* key_scale;
  uint8_t* value;
  float* value_scale;
  int8_t* bounds;
  float* bound_scale;
  int32_t kv_heads;
};

struct CacheMove {  // a write's inputs or a read's outputs
  Cache cache;
  CacheRows rows;
  InputTensor key, value;
  int32_t batch;
};

// How workgroups share out the pages of blocks of query rows: a workgroup per block; `parts` equal parts of each
// block (fewer where a part would have less than `least_share` pages); or equal shares of all blocks' pages in a line.
enum class CacheShares : int32_t { kWhole, kEven, kLine };

struct CachePieces {  // of a block: its first in the workspace, and how many; 1: the output is written
  int64_t first, parts;
};

// Pieces' sums [piece, row, D], maxima and totals [piece, row] and the blocks' pieces are in the workspace.
struct CacheAttention {
  Cache cache;
  CacheRows rows;
  InputTensor query;
  const uint8_t* mask;
  int64_t mask_stride_batch, mask_stride_row;
  const int32_t* selected;
  void* output;
  float scale;
  int32_t batch, heads, budget;
  CacheShares shares;
  int32_t parts, least_share, blocks_of_unit;
  int64_t workgroups;
  float* partial;
  float2* partial_stats;
  CachePieces* pieces;  // of each block
};

struct CacheParts {
  CacheShares shares;
  int64_t parts, least_share, blocks_of_unit, workgroups;
  int64_t rows, bytes;  // of the workspace
};

struct CacheSelect {
  Cache cache;
  CacheRows rows;
  InputTensor query;
  int32_t* output;
  float* scores;
  int32_t batch, heads, budget;
};

// Which instantiation a call takes.
struct CacheForm {
  bool bf16, fp8;
  int head_dim;
};

int64_t cache_select_scores(const CacheSelect& a, int cus);   // floats of the workspace
int64_t cache_select_most_workgroups(const CacheSelect& a);  // a launch takes no more, whichever kernel it is of

hipError_t launch_cache_write(const CacheMove& a, CacheForm form, hipStream_t stream);
hipError_t launch_cache_read(const CacheMove& a, CacheForm form, hipStream_t stream);
CacheParts cache_attention_parts(const CacheAttention& a, int head_dim, int cus);
hipError_t launch_cache_attention(const CacheAttention& a, CacheForm form, hipStream_t stream);
hipError_t launch_cache_select(const CacheSelect& a, CacheForm form, int cus, hipStream_t stream);

#ifdef __HIPCC__

// Calls f(integral_constant bf16, fp8, D) for a form.
template <typename F>
inline hipError_t with_cache_form(CacheForm form, F f) {
  const auto by_dim = [&](auto bf16, auto fp8) {
    return form.head_dim == 64 ? f(bf16, fp8, std::integral_constant<int, 64>{}) : f(bf16, fp8, std::integral_constant<int, 128>{});
  };
  const auto by_code = [&](auto bf16) { return form.fp8 ? by_dim(bf16, std::true_type{}) : by_dim(bf16, std::false_type{}); };
  return form.bf16 ? by_code(std::true_type{}) : by_code(std::false_type{});
}

template <bool kFp8>
__device__ __forceinline__ float code_value(uint32_t code) {  // the value of the code in the low byte
  if constexpr (kFp8) return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code), 0);
  return static_cast<float>(static_cast<int8_t>(code));
}

// How a row is held, from its largest magnitude `a` (NaN left out) and whether all of it is finite.
struct RowCode {
  float inv;    // values times this are rounded to codes
  float scale;  // a code stands for code * scale
};

template <bool kFp8>
__device__ __forceinline__ RowCode row_code(float a, bool finite) {
  constexpr float kLargest = kFp8 ? 448.0f : 127.0f;
  if (!finite) return RowCode{0.0f, __builtin_nanf("")};
  if (a < kTinyRow) return RowCode{0.0f, 0.0f};
  return RowCode{kLargest / a, a / kLargest};
}

// round_half_even(x * inv) as a byte.  |x * inv| is below L (1 + 2^-22): it rounds to at most L without a clamp.
// INT8: adding 1.5 * 2^23 rounds to an integer, whose two's complement the low mantissa bits hold.  A row of zero
// codes has inv = 0; its infinities and NaN give 0 all the same.
// The product is rounded before it is: a fused multiply-add would break other ties.
template <bool kFp8>
__device__ __forceinline__ uint32_t code_of_value(float x, float inv) {
#pragma clang fp contract(off)
  const float y = inv == 0.0f ? 0.0f : x * inv;
  if constexpr (kFp8) return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false)) & 0xffu;
  return __float_as_uint(y + kAccBiasValue) & 0xffu;
}

template <bool kBf16>
__device__ __forceinline__ float widen(uint16_t bits) {
  if constexpr (kBf16) return __uint_as_float(static_cast<uint32_t>(bits) << 16);
  return half_bits_to_float(bits);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (kBf16) return pack_bf16x2(a, b);
  return pack_half2(a, b);
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

#endif  // __HIPCC__

}  // namespace piper
