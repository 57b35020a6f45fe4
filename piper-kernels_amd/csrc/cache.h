// The quantised cache's addressing and value rules (include/piper_cache.h), shared by its kernels.  The index
// arithmetic is plain host and device code, so that the CPU tests run the very functions that keep the kernels
// inside their buffers.
#pragma once

#include <stdint.h>

#ifndef __HIPCC__
#define __host__
#define __device__
#endif

namespace piper {

constexpr int kPage = 64;
constexpr float kTinyRow = 0x1p-118f;  // rows below this are zeros: 448 / kTinyRow is finite

// Where a call's rows stand; see piper_cache_rows.
struct CacheRows {
  const int32_t* page_table;
  const int32_t* starts;
  const int32_t* counts;
  int64_t table_stride;
  int64_t pages;
  int32_t table_width;
  int32_t tokens;

  __host__ __device__ int64_t start(int64_t b) const { return starts[b]; }
  __host__ __device__ int count(int64_t b) const {
    const int n = counts != nullptr ? counts[b] : tokens;
    return n < 0 ? 0 : n > tokens ? tokens : n;
  }
  // The cache page of a sequence's `logical` page, or -1: the only way to a page, for every kernel.
  __host__ __device__ int64_t page(int64_t b, int64_t logical) const {
    if (logical < 0 || logical >= table_width) return -1;
    const int32_t p = page_table[b * table_stride + logical];
    return p >= 0 && p < pages ? p : -1;
  }
  // Positions [0, end) that row `i` and those before it can see: 0 where the row sees nothing.
  __host__ __device__ int64_t end(int64_t b, int64_t i) const {
    const int64_t last = start(b) + i + 1, room = static_cast<int64_t>(table_width) * kPage;
    return last < 0 ? 0 : last > room ? room : last;
  }
};

// The rows of a call that stand in a sequence's page `logical`: [first, first + n), row `first` in slot `slot`.
struct PageRows {
  int first, n, slot;
};

__host__ __device__ inline PageRows rows_in_page(const CacheRows& rows, int64_t b, int64_t logical) {
  const int64_t start = rows.start(b), count = rows.count(b), base = logical * kPage;
  const int64_t lo = start > base ? start : base;
  const int64_t hi = start + count < base + kPage ? start + count : base + kPage;
  if (logical < 0 || lo >= hi) return PageRows{0, 0, 0};
  return PageRows{static_cast<int>(lo - start), static_cast<int>(hi - lo), static_cast<int>(lo - base)};
}

// A call's rows of one sequence touch at most this many pages, from start / 64 (rounded down) on.
__host__ __device__ inline int64_t pages_touched(int64_t tokens) { return (tokens + kPage - 2) / kPage + 1; }

__host__ __device__ inline int64_t floor_page(int64_t position) {
  return position >= 0 ? position / kPage : -((kPage - 1 - position) / kPage);
}

// Byte of token `slot`, feature d in a page's values.
__host__ __device__ inline int value_offset(int slot, int d, int head_dim) {
  return (slot / 8) * head_dim * 8 + d * 8 + slot % 8;
}

}  // namespace piper
