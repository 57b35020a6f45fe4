// The quantised paged KV cache: writing, reading, page selection, and the C entry points (include/piper_cache.h).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cache_kernels.h"
#include "host.h"
#include "piper_cache.h"

namespace piper {
namespace {

// ---- write ----------------------------------------------------------------------------------------------------------

// One wave per page touched and K/V head: token by token, the row's largest magnitude over the lanes, then its codes.
template <bool kBf16, bool kFp8, int kDim>
__global__ __launch_bounds__(kWave) void cache_write_kernel(CacheMove a) {
  constexpr int kPer = kDim / kWave;  // features of a lane
  const int lane = threadIdx.x;
  const int64_t touched = pages_touched(a.rows.tokens);
  const int64_t unit = blockIdx.x / touched;
  const int64_t b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int64_t logical = floor_page(a.rows.start(b)) + blockIdx.x % touched;
  const PageRows in = rows_in_page(a.rows, b, logical);
  const int64_t page = a.rows.page(b, logical);
  if (in.n == 0 || page < 0) return;
  const int64_t record = page * a.cache.kv_heads + h;
  uint8_t* const keys = a.cache.key + record * kPage * kDim;
  uint8_t* const values = a.cache.value + record * kPage * kDim;
  const bool fills = in.slot + in.n == kPage;
  float upper[kPer], lower[kPer];
  for (int e = 0; e < kPer; ++e) upper[e] = -__builtin_inff(), lower[e] = __builtin_inff();

  for (int slot = fills ? 0 : in.slot; slot < in.slot + in.n; ++slot) {
    float k[kPer];
    if (slot < in.slot) {  // a full page's earlier keys, for its bounds
      const float s = a.cache.key_scale[record * kPage + slot];
      for (int e = 0; e < kPer; ++e) k[e] = code_value<kFp8>(keys[slot * kDim + lane * kPer + e]) * s;
    } else {
      const int64_t i = in.first + slot - in.slot;
      for (int part = 0; part < 2; ++part) {
        const InputTensor& t = part == 0 ? a.key : a.value;
        const uint16_t* row = static_cast<const uint16_t*>(t.data) + b * t.stride_batch + h * t.stride_head + i * t.stride_seq;
        float x[kPer], top = 0.0f;
        bool finite = true;
        for (int e = 0; e < kPer; ++e) {
          x[e] = widen<kBf16>(row[lane * kPer + e]);
          top = fmaxf(top, fabsf(x[e]));
          finite = finite && is_finite(x[e]);
        }
        const RowCode code = row_code<kFp8>(wave_max(top), __all(finite));
        for (int e = 0; e < kPer; ++e) {
          const uint32_t c = code_of_value<kFp8>(x[e], code.inv);
          if (part == 0) {
            keys[slot * kDim + lane * kPer + e] = static_cast<uint8_t>(c);
            k[e] = code_value<kFp8>(c) * code.scale;
          } else {
            values[value_offset(slot, lane * kPer + e, kDim)] = static_cast<uint8_t>(c);
          }
        }
        if (lane == 0) (part == 0 ? a.cache.key_scale : a.cache.value_scale)[record * kPage + slot] = code.scale;
      }
    }
    for (int e = 0; e < kPer; ++e) upper[e] = fmaxf(upper[e], k[e]), lower[e] = fminf(lower[e], k[e]);
  }
  if (!fills) return;
  float top = 0.0f;
  for (int e = 0; e < kPer; ++e) {
    if (upper[e] < lower[e]) upper[e] = lower[e] = 0.0f;  // every key of the page is NaN
    top = fmaxf(top, fmaxf(fabsf(upper[e]), fabsf(lower[e])));
  }
  const RowCode code = row_code<false>(wave_max(top), true);
  for (int e = 0; e < kPer; ++e) {
    a.cache.bounds[record * 2 * kDim + lane * kPer + e] = static_cast<int8_t>(code_of_value<false>(upper[e], code.inv));
    a.cache.bounds[record * 2 * kDim + kDim + lane * kPer + e] = static_cast<int8_t>(code_of_value<false>(lower[e], code.inv));
  }
  if (lane == 0) a.cache.bound_scale[record] = code.scale;
}

// ---- read -----------------------------------------------------------------------------------------------------------

// One thread per eight features of a row's key and value.
template <bool kBf16, bool kFp8, int kDim>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheMove a) {
  constexpr int kPieces = kDim / 8;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = at / kPieces;
  const int piece = static_cast<int>(at % kPieces);
  const int64_t i = row % a.rows.tokens, unit = row / a.rows.tokens;
  const int64_t b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  if (b >= a.batch) return;
  const int64_t position = a.rows.start(b) + i;
  const int64_t page = i < a.rows.count(b) && position >= 0 ? a.rows.page(b, position / kPage) : -1;
  uint32_t key[4] = {}, value[4] = {};
  if (page >= 0) {
    const int64_t record = page * a.cache.kv_heads + h;
    const int slot = static_cast<int>(position % kPage);
    const float ks = a.cache.key_scale[record * kPage + slot], vs = a.cache.value_scale[record * kPage + slot];
    const uint8_t* k = a.cache.key + record * kPage * kDim + slot * kDim + piece * 8;
    const uint8_t* v = a.cache.value + record * kPage * kDim + value_offset(slot, piece * 8, kDim);
    for (int e = 0; e < 4; ++e) {
      key[e] = narrow2<kBf16>(code_value<kFp8>(k[2 * e]) * ks, code_value<kFp8>(k[2 * e + 1]) * ks);
      value[e] = narrow2<kBf16>(code_value<kFp8>(v[16 * e]) * vs, code_value<kFp8>(v[16 * e + 8]) * vs);
    }
  }
  const_cast<uint4*>(static_cast<const uint4*>(a.key.data))[at] = uint4{key[0], key[1], key[2], key[3]};
  const_cast<uint4*>(static_cast<const uint4*>(a.value.data))[at] = uint4{value[0], value[1], value[2], value[3]};
}

// ---- selection ------------------------------------------------------------------------------------------------------

// Scores of a row's earlier pages: one workgroup per row and K/V head, a thread per page.
template <bool kBf16, int kDim>
__global__ __launch_bounds__(256) void cache_score_kernel(CacheSelect a) {
  __shared__ int8_t codes[2 * kDim];  // q+ beside the upper bound, q- beside the lower one
  __shared__ float scale;
  const int64_t row = blockIdx.x;
  const int64_t i = row % a.rows.tokens, unit = row / a.rows.tokens;
  const int64_t b = unit / a.cache.kv_heads, h = unit % a.cache.kv_heads;
  const int64_t end = a.rows.end(b, i);
  const int group = a.heads / a.cache.kv_heads;
  const int earlier = i < a.rows.count(b) && end > 0 ? static_cast<int>((end - 1) / kPage) : 0;
  float* const scores = a.scores + row * a.rows.table_width;
  for (int g = 0; g < group; ++g) {
    __syncthreads();
    if (threadIdx.x < kWave) {
      const uint16_t* q = static_cast<const uint16_t*>(a.query.data) + b * a.query.stride_batch +
                          (h * group + g) * a.query.stride_head + i * a.query.stride_seq;
      float x[kDim / kWave], top = 0.0f;
      bool finite = true;
      for (int e = 0; e < kDim / kWave; ++e) {
        x[e] = widen<kBf16>(q[threadIdx.x + e * kWave]);
        top = fmaxf(top, fabsf(x[e]));
        finite = finite && is_finite(x[e]);
      }
      const RowCode code = row_code<false>(wave_max(top), __all(finite));
      for (int e = 0; e < kDim / kWave; ++e) {
        const int8_t c = static_cast<int8_t>(code_of_value<false>(x[e], code.inv));
        codes[threadIdx.x + e * kWave] = c > 0 ? c : 0;
        codes[kDim + threadIdx.x + e * kWave] = c < 0 ? c : 0;
      }
      if (threadIdx.x == 0) scale = code.scale;
    }
    __syncthreads();
    for (int p = threadIdx.x; p < earlier; p += 256) {
      const int64_t page = a.rows.page(b, p);
      const int64_t record = page * a.cache.kv_heads + h;
      float score = -__builtin_inff();
      if (page >= 0) {
        int dot = 0;
        for (int d = 0; d < 2 * kDim; ++d) dot += static_cast<int>(a.cache.bounds[record * 2 * kDim + d]) * codes[d];
        score = __fmul_rn(static_cast<float>(dot), scale);
      }
      if (g > 0) score = fmaxf(score, scores[p]);
      if (g == group - 1 && page >= 0) score = __fmul_rn(score, a.cache.bound_scale[record]);
      scores[p] = score;
    }
  }
}

// Scores in the order of whole numbers: the larger the score, the larger the number (-0 is 0).
__device__ __forceinline__ uint32_t score_order(float score) {
  const uint32_t u = __float_as_uint(score + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The budget - 1 best earlier pages of a row: the last one's score found eight bits at a time by counting, then the
// pages above it, and the first of those at it, in their order.
__global__ __launch_bounds__(256) void cache_select_kernel(CacheSelect a) {
  __shared__ int counts[256];
  __shared__ int found[2];
  __shared__ int wave_above[4], wave_at[4];
  const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
  const int64_t row = blockIdx.x;
  const int64_t i = row % a.rows.tokens, unit = row / a.rows.tokens;
  const int64_t b = unit / a.cache.kv_heads;
  const int64_t end = a.rows.end(b, i);
  int32_t* const out = a.output + row * a.budget;
  // a row that is none, or stands where the table does not reach
  const bool real = i < a.rows.count(b) && end > 0 && end == a.rows.start(b) + i + 1;
  const int own = real ? static_cast<int>((end - 1) / kPage) : -1;
  const int earlier = own > 0 ? own : 0;
  const int taken = earlier < a.budget - 1 ? earlier : a.budget - 1;
  const float* const scores = a.scores + row * a.rows.table_width;
  uint32_t prefix = 0;
  int left = taken;  // pages still to take among those that share the prefix
  if (taken < earlier && taken > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      counts[thread] = 0;
      __syncthreads();
      for (int p = thread; p < earlier; p += 256) {
        const uint32_t u = score_order(scores[p]);
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&counts[(u >> shift) & 255u], 1);
      }
      __syncthreads();
      if (thread == 0) {
        int digit = 255, more = left;
        while (counts[digit] < more) more -= counts[digit--];
        found[0] = digit;
        found[1] = more;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(found[0]) << shift;
      left = found[1];
      __syncthreads();
    }
  }
  int done = 0, at_done = 0;  // pages taken so far, and how many of them at the last score
  for (int base = 0; base < earlier && taken > 0; base += 256) {
    const int p = base + thread;
    const uint32_t u = p < earlier ? score_order(scores[p]) : 0;
    const bool all = taken == earlier;
    const bool above = p < earlier && (all || u > prefix), at = p < earlier && !all && u == prefix;
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t at_lanes = __ballot(at);
    if (lane == 0) wave_at[wave] = __popcll(at_lanes);
    __syncthreads();
    int rank = at_done + __popcll(at_lanes & below);
    for (int w = 0; w < 4; ++w) rank += w < wave ? wave_at[w] : 0, at_done += wave_at[w];
    const bool take = above || (at && rank < left);
    const uint64_t lanes = __ballot(take);
    if (lane == 0) wave_above[wave] = __popcll(lanes);
    __syncthreads();
    int place = done + __popcll(lanes & below);
    for (int w = 0; w < 4; ++w) place += w < wave ? wave_above[w] : 0, done += wave_above[w];
    if (take) out[place] = p;
    __syncthreads();
  }
  if (thread == 0 && real) out[taken] = own;
  for (int p = taken + (real ? 1 : 0) + thread; p < a.budget; p += 256) out[p] = -1;
}

}  // namespace

hipError_t launch_cache_write(const CacheMove& a, CacheForm form, hipStream_t stream) {
  const int64_t blocks = a.batch * a.cache.kv_heads * pages_touched(a.rows.tokens);
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    cache_write_kernel<decltype(bf16)::value, decltype(fp8)::value, decltype(dim)::value>
        <<<dim3(static_cast<uint32_t>(blocks)), dim3(kWave), 0, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_cache_read(const CacheMove& a, CacheForm form, hipStream_t stream) {
  const int64_t threads = static_cast<int64_t>(a.batch) * a.cache.kv_heads * a.rows.tokens * (form.head_dim / 8);
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    cache_read_kernel<decltype(bf16)::value, decltype(fp8)::value, decltype(dim)::value>
        <<<dim3(static_cast<uint32_t>(ceil_div(threads, 256))), dim3(256), 0, stream>>>(a);
    return hipGetLastError();
  });
}

int64_t cache_select_scores(const CacheSelect& a) {
  return a.budget > 1 ? static_cast<int64_t>(a.batch) * a.cache.kv_heads * a.rows.tokens * a.rows.table_width : 0;
}

hipError_t launch_cache_select(const CacheSelect& a, CacheForm form, hipStream_t stream) {
  const dim3 blocks(static_cast<uint32_t>(static_cast<int64_t>(a.batch) * a.cache.kv_heads * a.rows.tokens));
  form.fp8 = false;  // the bounds are INT8 in every cache
  return with_cache_form(form, [&](auto bf16, auto, auto dim) {
    if (a.budget > 1) {
      cache_score_kernel<decltype(bf16)::value, decltype(dim)::value><<<blocks, dim3(256), 0, stream>>>(a);
      if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    cache_select_kernel<<<blocks, dim3(256), 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace piper

// ---- C entry points --------------------------------------------------------------------------------------------------

namespace {

using piper::aligned16;
using piper::fail;

constexpr int64_t kMaxBlocks = int64_t(1) << 30;  // of a launch; grids are 32-bit

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
  // pages and widths are int32 in the kernels, as table entries are; a grid has at most kMaxBlocks workgroups
  if (c.pages > INT32_MAX || r.table_width > (1 << 24) || r.tokens > (1 << 26) || c.kv_heads > (1 << 16) || r.batch > (1 << 24) ||
      r.batch * c.kv_heads > kMaxBlocks / r.tokens)
    return fail(PIPER_ERROR_UNSUPPORTED, "cache call too large for this build");
  return PIPER_OK;
}

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
  if (!aligned16(c.bounds) || !aligned16(c.bound_scale)) return fail(PIPER_ERROR_INVALID_ARGUMENT, "cache arrays must be 16-byte aligned");
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
  if (heads > (1 << 20) || r.batch * heads > kMaxBlocks / r.tokens) return fail(PIPER_ERROR_UNSUPPORTED, "cache call too large for this build");
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
  *bytes = piper::cache_attention_parts(attention_of(*a), a->cache.head_dim, cus).bytes;
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
  if (parts.workgroups > kMaxBlocks) return fail(PIPER_ERROR_UNSUPPORTED, "cache call too large for this build");
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
  *bytes = 4 * piper::cache_select_scores(select_of(*a));
  return PIPER_OK;
}

extern "C" int piper_cache_select(const piper_cache_select_args* a, void* stream) {
  if (int st = check_select(a)) return st;
  if (int st = check_rows(a->rows)) return st;
  if (int st = check_bounds(a->cache)) return st;
  if (int st = check_tensor("query", a->query)) return st;
  if (a->output == nullptr) return fail(PIPER_ERROR_INVALID_ARGUMENT, "output pointer is NULL");
  const piper::CacheSelect select = select_of(*a);
  if (int st = check_workspace(a->workspace, a->workspace_bytes, 4 * piper::cache_select_scores(select))) return st;
  return launched(piper::launch_cache_select(select, form_of(a->cache, a->dtype), static_cast<hipStream_t>(stream)), "cache select");
}
