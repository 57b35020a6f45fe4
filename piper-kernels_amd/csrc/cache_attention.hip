// Attention over the quantised paged cache (include/piper_cache.h).
#include <type_traits>

#include "cache_kernels.h"

namespace piper {
namespace {

// One wave per query row: a page's 64 scores over its lanes, the running maximum and sum of the softmax, then the
// page's values feature by feature.
template <bool kBf16, bool kFp8, int kDim>
__global__ __launch_bounds__(kWave) void cache_attention_kernel(CacheAttention a) {
  constexpr int kPer = kDim / kWave;
  __shared__ float query[kDim];
  __shared__ float weight[kPage];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;  // [batch, heads, tokens]
  const int64_t i = row % a.rows.tokens, hq = row / a.rows.tokens % a.heads, b = row / a.rows.tokens / a.heads;
  const int64_t h = hq / (a.heads / a.cache.kv_heads);
  const int64_t start = a.rows.start(b);
  const int count = a.rows.count(b);
  uint16_t* const out = static_cast<uint16_t*>(a.output) + row * kDim;

  const uint16_t* q = static_cast<const uint16_t*>(a.query.data) + b * a.query.stride_batch + hq * a.query.stride_head + i * a.query.stride_seq;
  for (int e = 0; e < kPer; ++e) query[lane * kPer + e] = widen<kBf16>(q[lane * kPer + e]);
  __syncthreads();

  // a masked row can see every drafted token, any other what stands before it
  const int64_t end = i >= count ? 0 : a.rows.end(b, a.mask != nullptr ? count - 1 : i);
  const int64_t pages = (end + kPage - 1) / kPage;
  const int32_t* const selected =
      a.selected != nullptr ? a.selected + ((b * a.cache.kv_heads + h) * a.rows.tokens + i) * a.budget : nullptr;
  const int64_t steps = selected != nullptr ? a.budget : pages;
  const float factor = a.scale * kLog2e;
  float top = -__builtin_inff(), total = 0.0f, sum[kPer] = {};
  for (int64_t step = 0; step < steps; ++step) {
    const int64_t logical = selected != nullptr ? selected[step] : step;
    const int64_t page = logical < pages ? a.rows.page(b, logical) : -1;
    if (page < 0) continue;
    const int64_t record = page * a.cache.kv_heads + h;
    const int64_t position = logical * kPage + lane;
    bool visible = position < end;
    if (a.mask != nullptr && position >= start)
      visible = visible && a.mask[b * a.mask_stride_batch + i * a.mask_stride_row + (position - start)] != 0;
    float s = -__builtin_inff();
    if (visible) {
      const uint8_t* k = a.cache.key + (record * kPage + lane) * kDim;
      s = 0.0f;
      for (int d = 0; d < kDim; ++d) s = fmaf(query[d], code_value<kFp8>(k[d]), s);
      s *= a.cache.key_scale[record * kPage + lane] * factor;
    }
    if (!__any(visible)) continue;
    const float next = fmaxf(top, wave_max(s));
    const float base = next == -__builtin_inff() ? 0.0f : next;
    const float p = visible ? exp2f(s - base) : 0.0f;
    const float keep = exp2f(top - base);
    top = next;
    float p_sum = p;
    for (int m = 32; m > 0; m >>= 1) p_sum += __shfl_xor(p_sum, m, 64);
    total = total * keep + p_sum;
    weight[lane] = visible ? p * a.cache.value_scale[record * kPage + lane] : 0.0f;
    __syncthreads();
    for (int e = 0; e < kPer; ++e) sum[e] *= keep;
    for (int slot = 0; slot < kPage; ++slot) {
      const float w = weight[slot];
      if (w == 0.0f) continue;  // nothing that is not seen is read, whatever its bytes stand for
      for (int e = 0; e < kPer; ++e)
        sum[e] = fmaf(w, code_value<kFp8>(a.cache.value[record * kPage * kDim + value_offset(slot, lane * kPer + e, kDim)]), sum[e]);
    }
    __syncthreads();
  }
  for (int e = 0; e < kPer; ++e) {
    const float o = total == 0.0f ? 0.0f : sum[e] / total;
    out[lane * kPer + e] = static_cast<uint16_t>(narrow2<kBf16>(o, 0.0f));
  }
}

}  // namespace

hipError_t launch_cache_attention(const CacheAttention& a, CacheForm form, hipStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(a.batch) * a.heads * a.rows.tokens;
  return with_cache_form(form, [&](auto bf16, auto fp8, auto dim) {
    cache_attention_kernel<decltype(bf16)::value, decltype(fp8)::value, decltype(dim)::value>
        <<<dim3(static_cast<uint32_t>(blocks)), dim3(kWave), 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace piper
