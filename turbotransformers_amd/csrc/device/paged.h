// What the kernels over a cache in pages share: the arguments as the device sees them, their checks, which sequence a row belongs to.
#pragma once

#include <algorithm>

#include "common.h"

namespace ttmi {

struct PagedView {
  const int32_t* table;
  const int32_t* starts;
  const int32_t* lengths;
  int* error;
  int64_t table_pitch;
  int batch, tokens, pages, kv_heads, page_shift;
  int head_dim;
};

// Positions and rows are held in 32 bits, offsets into the cache in 64.
inline int paged_view(const ttmi_paged_cache* cache, const ttmi_paged_batch* batch, int64_t heads, PagedView* out) {
  constexpr int64_t kMost = INT32_MAX;
  TTMI_REQUIRE(cache != nullptr && batch != nullptr, "cache or batch is null");
  TTMI_REQUIRE(cache->page_size >= 1 && cache->page_size <= 4096 && (cache->page_size & (cache->page_size - 1)) == 0,
               "page_size must be a power of two up to 4096");
  TTMI_REQUIRE(cache->head_dim >= 16 && cache->head_dim <= 256 && cache->head_dim % 16 == 0, "head_dim must be a multiple of 16 up to 256");
  TTMI_REQUIRE(cache->kv_heads >= 1 && cache->kv_heads <= 65535 && heads >= 1 && heads <= 65535 && heads % cache->kv_heads == 0,
               "heads must be a multiple of kv_heads, at most 65535");
  TTMI_REQUIRE(cache->pages >= 0 && cache->pages <= kMost && batch->table_pitch >= 0 && batch->table_pitch <= (1 << 30) / cache->page_size,
               "too many pages: positions must not pass 2^30");
  TTMI_REQUIRE(batch->batch >= 0 && batch->batch <= kMost / 2 && batch->tokens >= 0 && batch->tokens <= kMost / 256, "batch is too large");
  if (batch->batch > 0 && batch->tokens > 0) {
    TTMI_REQUIRE(batch->starts != nullptr && batch->lengths != nullptr && (batch->table != nullptr || batch->table_pitch == 0),
                 "starts, lengths or table is null");
    TTMI_REQUIRE(cache->pages == 0 || (cache->keys != nullptr && cache->values != nullptr), "the cache's keys or values are null");
    TTMI_REQUIRE(((reinterpret_cast<uintptr_t>(cache->keys) | reinterpret_cast<uintptr_t>(cache->values)) & 15) == 0,
                 "the cache's keys and values must be 16-byte aligned");
  }
  out->table = batch->table, out->starts = batch->starts, out->lengths = batch->lengths, out->error = async_error_flag();
  out->table_pitch = cache->pages > 0 ? batch->table_pitch : 0;  // (without pages every key is one too many)
  out->batch = (int)batch->batch, out->tokens = (int)batch->tokens, out->pages = (int)cache->pages, out->kv_heads = (int)cache->kv_heads;
  out->page_shift = __builtin_ctzll((unsigned long long)cache->page_size), out->head_dim = (int)cache->head_dim;
  return 0;
}

inline bool rows_aligned(const void* p, int64_t pitch, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch * (int64_t)dtype_size(dtype) % 16 == 0;
}

__device__ __forceinline__ void page_error(const PagedView& view) {
  if (view.error != nullptr) *view.error = kPageOutOfRange;
}

// The number of sequences whose rows end at or before `row` (uniform over the wavefront): the sequence the row belongs to, or `batch`
// behind the last one.  Every lane looks at one sequence of 64: two trips to memory for batches of up to 64, where a search by halves takes six.
__device__ __forceinline__ int sequence_of(const PagedView& view, int row) {
  const int lane = (int)(threadIdx.x % kWave);
  int found = 0;
  for (int base = 0; base < view.batch; base += kWave) {
    const bool before = base + lane < view.batch && view.starts[base + lane + 1] <= row;
    const int n = __popcll(__ballot(before));
    found += n;
    if (n < kWave) break;
  }
  return __builtin_amdgcn_readfirstlane(found);
}

}  // namespace ttmi
