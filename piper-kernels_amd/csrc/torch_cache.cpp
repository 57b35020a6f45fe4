// The cache operators' torch kernels (libpiper_torch.so): piper_kernels::cache_write, cache_read, cache_attention
// and cache_select on GPU tensors, over the C ABI of include/piper_cache.h.  The ops' definitions and fakes are
// in Python (attention/quantized_cache/hip.py).  Everything the kernels rely on is checked here, before anything is
// launched: the public functions call these at once and look for the words of a refusal only after one (a good call's
// checks take 10 us in Python, as long as a short call's kernels).
#include <optional>

#include "piper_cache.h"
#include "torch_common.h"

namespace {

using at::Tensor;
using piper_torch::check;
using piper_torch::dtype_code;
using piper_torch::native_input;
using piper_torch::tensor_arg;

// The current stream of a device, current for the guard's lifetime.
struct Place {
  c10::OptionalDeviceGuard guard;
  c10::Device device;
  c10::Stream stream;
  void* handle;

  explicit Place(const Tensor& t)
      : guard(t.device()),
        device(t.device()),
        stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index())),
        handle(static_cast<hipStream_t>(c10::hip::HIPStreamMasqueradingAsCUDA(stream))) {}

  // the caching allocator must not hand a tensor's memory to another stream before this one is done with it
  void keep(const Tensor& t) const { t.record_stream(stream); }
  void keep(const std::optional<Tensor>& t) const {
    if (t.has_value()) keep(*t);
  }
};

void check_dense(const Tensor& t, const Place& place, const char* name) {
  TORCH_CHECK(t.device() == place.device, "piper_kernels: ", name, " must be on ", place.device, ", got ", t.device());
  TORCH_CHECK(t.is_contiguous(), "piper_kernels: ", name, " must be contiguous");
}

// A cache's codes and scales, from the key codes' shape [pages, kv_heads, 64, D].
piper_cache codes_arg(const Place& place, const Tensor& key, const Tensor& key_scale, const Tensor& value, const Tensor& value_scale) {
  TORCH_CHECK(key.dim() == 4 && key.size(2) == PIPER_CACHE_PAGE, "piper_kernels: cache key must have shape [pages, kv_heads, 64, head_dim], got ",
              key.sizes());
  const int64_t p = key.size(0), h = key.size(1), d = key.size(3);
  TORCH_CHECK(value.sizes() == at::IntArrayRef({p, h, 8, d, 8}) && key_scale.sizes() == at::IntArrayRef({p, h, 64}) &&
                  value_scale.sizes() == at::IntArrayRef({p, h, 64}),
              "piper_kernels: the cache's arrays do not belong together, got ", key.sizes(), ", ", key_scale.sizes(), ", ", value.sizes(),
              " and ", value_scale.sizes());
  TORCH_CHECK((key.scalar_type() == at::kChar || key.scalar_type() == at::kFloat8_e4m3fn) && value.scalar_type() == key.scalar_type() &&
                  key_scale.scalar_type() == at::kFloat && value_scale.scalar_type() == at::kFloat,
              "piper_kernels: cache codes must use int8 or float8_e4m3fn and their scales float32");
  check_dense(key, place, "cache key");
  check_dense(key_scale, place, "cache key_scale");
  check_dense(value, place, "cache value");
  check_dense(value_scale, place, "cache value_scale");
  piper_cache c{};
  c.key = const_cast<void*>(key.const_data_ptr());
  c.key_scale = const_cast<float*>(key_scale.const_data_ptr<float>());
  c.value = const_cast<void*>(value.const_data_ptr());
  c.value_scale = const_cast<float*>(value_scale.const_data_ptr<float>());
  c.pages = p;
  c.kv_heads = h;
  c.head_dim = static_cast<int32_t>(d);
  c.code = key.scalar_type() == at::kChar ? PIPER_CACHE_INT8 : PIPER_CACHE_FP8;
  return c;
}

// Adds the bounds [pages, kv_heads, 2, D] to a cache (which has its sizes from them if it has none).
void bounds_arg(const Place& place, piper_cache& c, const Tensor& bounds, const Tensor& bound_scale) {
  TORCH_CHECK(bounds.dim() == 4 && bounds.size(2) == 2, "piper_kernels: cache bounds must have shape [pages, kv_heads, 2, head_dim], got ",
              bounds.sizes());
  if (c.pages == 0) {
    c.pages = bounds.size(0);
    c.kv_heads = bounds.size(1);
    c.head_dim = static_cast<int32_t>(bounds.size(3));
  }
  TORCH_CHECK(bounds.sizes() == at::IntArrayRef({c.pages, c.kv_heads, 2, c.head_dim}) && bound_scale.sizes() == at::IntArrayRef({c.pages, c.kv_heads}),
              "piper_kernels: the cache's arrays do not belong together, got ", bounds.sizes(), " and ", bound_scale.sizes());
  TORCH_CHECK(bounds.scalar_type() == at::kChar && bound_scale.scalar_type() == at::kFloat,
              "piper_kernels: cache bounds must use int8 and their scale float32");
  check_dense(bounds, place, "cache bounds");
  check_dense(bound_scale, place, "cache bound_scale");
  c.bounds = const_cast<int8_t*>(bounds.const_data_ptr<int8_t>());
  c.bound_scale = const_cast<float*>(bound_scale.const_data_ptr<float>());
}

piper_cache_rows rows_arg(const Place& place, const Tensor& table, const Tensor& starts, const std::optional<Tensor>& counts, int64_t batch,
                          int64_t tokens) {
  const auto whole = [&](const Tensor& t, int64_t dims, const char* name) {
    TORCH_CHECK(t.dim() == dims && t.size(0) == batch && t.scalar_type() == at::kInt && t.device() == place.device &&
                    (t.stride(dims - 1) == 1 || t.size(dims - 1) == 1),
                "piper_kernels: ", name, " must be an int32 tensor of ", batch, " rows on ", place.device, " with contiguous rows");
  };
  whole(table, 2, "page_table");
  whole(starts, 1, "starts");
  if (counts.has_value()) whole(*counts, 1, "counts");
  piper_cache_rows r{};
  r.page_table = table.const_data_ptr<int32_t>();
  r.starts = starts.const_data_ptr<int32_t>();
  r.counts = counts.has_value() ? counts->const_data_ptr<int32_t>() : nullptr;
  r.table_stride = table.stride(0);
  r.table_width = table.size(1);
  r.batch = batch;
  r.tokens = tokens;
  return r;
}

void check_rows_tensor(const Place& place, const Tensor& t, const char* name, int64_t head_dim) {
  TORCH_CHECK(t.dim() == 4 && t.size(3) == head_dim && t.stride(3) == 1 && t.numel() > 0 && t.device() == place.device, "piper_kernels: ", name,
              " must have shape [batch, heads, tokens, ", head_dim, "] and a contiguous head dimension on ", place.device, ", got ", t.sizes());
}

Tensor workspace_of(const Tensor& like, int64_t bytes) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

void cache_write(const Tensor& key, const Tensor& value, const Tensor& cache_key, const Tensor& cache_key_scale, const Tensor& cache_value,
                 const Tensor& cache_value_scale, const Tensor& cache_bounds, const Tensor& cache_bound_scale, const Tensor& page_table,
                 const Tensor& starts, const std::optional<Tensor>& counts) {
  const Place place(cache_key);
  piper_cache_write_args a{};
  a.abi_version = PIPER_CACHE_ABI_VERSION;
  a.cache = codes_arg(place, cache_key, cache_key_scale, cache_value, cache_value_scale);
  bounds_arg(place, a.cache, cache_bounds, cache_bound_scale);
  check_rows_tensor(place, key, "key", a.cache.head_dim);
  check_rows_tensor(place, value, "value", a.cache.head_dim);
  TORCH_CHECK(key.sizes() == value.sizes() && key.size(1) == a.cache.kv_heads && key.scalar_type() == value.scalar_type(),
              "piper_kernels: key and value must agree and have the cache's heads, got ", key.sizes(), " and ", value.sizes());
  a.dtype = dtype_code(key);
  a.rows = rows_arg(place, page_table, starts, counts, key.size(0), key.size(2));
  const Tensor k = native_input(key), v = native_input(value);
  a.key = tensor_arg(k);
  a.value = tensor_arg(v);
  check(piper_cache_write(&a, place.handle), "piper_cache_write");
  for (const Tensor* t : {&k, &v, &cache_key, &cache_key_scale, &cache_value, &cache_value_scale, &cache_bounds, &cache_bound_scale, &page_table,
                          &starts})
    place.keep(*t);
  place.keep(counts);
}

std::tuple<Tensor, Tensor> cache_read(const Tensor& cache_key, const Tensor& cache_key_scale, const Tensor& cache_value,
                                      const Tensor& cache_value_scale, const Tensor& page_table, const Tensor& starts,
                                      const std::optional<Tensor>& counts, int64_t size, at::ScalarType dtype) {
  const Place place(cache_key);
  piper_cache_read_args a{};
  a.abi_version = PIPER_CACHE_ABI_VERSION;
  a.dtype = dtype_code(dtype);
  a.cache = codes_arg(place, cache_key, cache_key_scale, cache_value, cache_value_scale);
  TORCH_CHECK(page_table.dim() == 2 && size > 0, "piper_kernels: page_table must have shape [batch, pages] and size be positive");
  a.rows = rows_arg(place, page_table, starts, counts, page_table.size(0), size);
  const auto options = cache_key.options().dtype(dtype);
  Tensor key = at::empty({a.rows.batch, a.cache.kv_heads, size, a.cache.head_dim}, options), value = at::empty_like(key);
  a.key = key.mutable_data_ptr();
  a.value = value.mutable_data_ptr();
  check(piper_cache_read(&a, place.handle), "piper_cache_read");
  for (const Tensor* t : {&cache_key, &cache_key_scale, &cache_value, &cache_value_scale, &page_table, &starts}) place.keep(*t);
  place.keep(counts);
  return {std::move(key), std::move(value)};
}

Tensor cache_attention(const Tensor& query, const Tensor& cache_key, const Tensor& cache_key_scale, const Tensor& cache_value,
                       const Tensor& cache_value_scale, const Tensor& page_table, const Tensor& starts, const std::optional<Tensor>& counts,
                       const std::optional<Tensor>& mask, const std::optional<Tensor>& selected, double scale) {
  const Place place(query);
  piper_cache_attention_args a{};
  a.abi_version = PIPER_CACHE_ABI_VERSION;
  a.dtype = dtype_code(query);
  a.scale = static_cast<float>(scale);
  a.cache = codes_arg(place, cache_key, cache_key_scale, cache_value, cache_value_scale);
  check_rows_tensor(place, query, "query", a.cache.head_dim);
  const int64_t batch = query.size(0), tokens = query.size(2);
  a.heads = query.size(1);
  a.rows = rows_arg(place, page_table, starts, counts, batch, tokens);
  const Tensor q = native_input(query);
  a.query = tensor_arg(q);
  Tensor seen, pages;
  if (mask.has_value()) {
    TORCH_CHECK(mask->dim() == 3 && (mask->size(0) == batch || mask->size(0) == 1) && mask->size(1) == tokens && mask->size(2) == tokens &&
                    mask->scalar_type() == at::kBool && mask->device() == place.device,
                "piper_kernels: mask must be a bool tensor [batch or 1, tokens, tokens] on ", place.device, ", got ", mask->sizes());
    seen = mask->stride(2) == 1 || tokens == 1 ? *mask : mask->contiguous();
    a.mask = static_cast<const uint8_t*>(seen.const_data_ptr());
    a.mask_stride_batch = seen.size(0) == 1 ? 0 : seen.stride(0);
    a.mask_stride_row = seen.stride(1);
  }
  if (selected.has_value()) {
    TORCH_CHECK(selected->dim() == 4 && selected->size(0) == batch && selected->size(1) == a.cache.kv_heads && selected->size(2) == tokens &&
                    selected->size(3) > 0 && selected->scalar_type() == at::kInt && selected->device() == place.device,
                "piper_kernels: selected must be an int32 tensor [batch, kv_heads, tokens, budget] on ", place.device, ", got ", selected->sizes());
    pages = selected->contiguous();
    a.selected = pages.const_data_ptr<int32_t>();
    a.budget = pages.size(3);
  }
  Tensor output = at::empty(query.sizes(), query.options().memory_format(at::MemoryFormat::Contiguous));
  a.output = output.mutable_data_ptr();
  int64_t bytes = 0;
  check(piper_cache_attention_workspace_bytes(&a, &bytes), "piper_cache_attention_workspace_bytes");
  const Tensor workspace = workspace_of(query, bytes);
  a.workspace = bytes > 0 ? workspace.mutable_data_ptr() : nullptr;
  a.workspace_bytes = bytes;
  check(piper_cache_attention(&a, place.handle), "piper_cache_attention");
  for (const Tensor* t : {&q, &cache_key, &cache_key_scale, &cache_value, &cache_value_scale, &page_table, &starts}) place.keep(*t);
  place.keep(counts);
  if (seen.defined()) place.keep(seen);
  if (pages.defined()) place.keep(pages);
  return output;
}

Tensor cache_select(const Tensor& query, const Tensor& cache_bounds, const Tensor& cache_bound_scale, const Tensor& page_table,
                    const Tensor& starts, const std::optional<Tensor>& counts, int64_t budget) {
  const Place place(query);
  piper_cache_select_args a{};
  a.abi_version = PIPER_CACHE_ABI_VERSION;
  a.dtype = dtype_code(query);
  bounds_arg(place, a.cache, cache_bounds, cache_bound_scale);
  check_rows_tensor(place, query, "query", a.cache.head_dim);
  a.heads = query.size(1);
  a.rows = rows_arg(place, page_table, starts, counts, query.size(0), query.size(2));
  const Tensor q = native_input(query);
  a.query = tensor_arg(q);
  a.budget = budget;
  int64_t bytes = 0;
  check(piper_cache_select_workspace_bytes(&a, &bytes), "piper_cache_select_workspace_bytes");
  Tensor output = at::empty({query.size(0), a.cache.kv_heads, query.size(2), budget}, query.options().dtype(at::kInt));
  const Tensor workspace = workspace_of(query, bytes);
  a.output = output.mutable_data_ptr<int32_t>();
  a.workspace = bytes > 0 ? workspace.mutable_data_ptr() : nullptr;
  a.workspace_bytes = bytes;
  check(piper_cache_select(&a, place.handle), "piper_cache_select");
  for (const Tensor* t : {&q, &cache_bounds, &cache_bound_scale, &page_table, &starts}) place.keep(*t);
  place.keep(counts);
  return output;
}

}  // namespace

void piper_torch::register_cache_kernels(torch::Library& library) {
  library.impl("cache_write", &cache_write);
  library.impl("cache_read", &cache_read);
  library.impl("cache_attention", &cache_attention);
  library.impl("cache_select", &cache_select);
}
