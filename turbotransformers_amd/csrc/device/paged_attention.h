// What the kernels of attention over pages share: their arguments, which keys a row sees and which part of them is whose, where rows of the cache lie.
//
// The rows of one sequence and key/value head are its new tokens' query heads of that group, token by token: row r is head r % group of the group, token
// r / group, so a tile of rows reads each key and value once for all heads that share it.
#pragma once

#include "attention_common.h"
#include "paged.h"

namespace ttmi {

constexpr int kFewRows = 16;  // rows of a sequence and key/value head that are the few-rows kernel's

struct PagedArgs {
  const void *q, *keys, *values;
  void* out;
  int64_t q_pitch, out_pitch;
  PagedView view;
  int heads, group, causal, window;  // window 0: none
  float scale_log2e;
  // Keys are cut at multiples of `chunk` (a multiple of 64), counted from the first of the sequence, into at most `splits` parts (the grid); a sequence that has more
  // keys than that takes longer parts.
  int chunk, splits;
  int every;  // the few-rows kernel takes sequences of any number of rows: the other one is not launched
  // rows whose keys lie in several parts: their sums [row][part][d] and, behind all of them, maxima and sums of the probabilities [row][part][2]
  float* partial;
  int64_t partial_rows;
};

struct Reach {
  int begin, end;  // keys
};
struct Sequence {
  int start, tokens, length, first;  // its first row, new tokens, keys, position of the first new token
  __device__ __forceinline__ Reach reach(const PagedArgs& a, int token) const {
    const int position = first + token;
    Reach r;
    r.begin = a.window > 0 ? max(0, position - a.window + 1) : 0;
    r.end = a.causal ? max(0, min(length, position + 1)) : length;
    if (r.begin >= r.end) r.begin = r.end = 0;
    return r;
  }
  // keys of a part
  __device__ __forceinline__ int chunk(const PagedArgs& a) const {
    return a.splits <= 1 ? INT32_MAX : max(a.chunk, ((length + a.splits - 1) / a.splits + 63) & ~63);
  }
};
__device__ __forceinline__ Sequence sequence(const PagedArgs& a, int b) {
  Sequence s;
  s.start = max(0, a.view.starts[b]);
  const int end = min(a.view.starts[b + 1], a.view.tokens), length = a.view.lengths[b];
  s.tokens = max(0, end - s.start);
  s.first = length - s.tokens;
  s.length = max(0, (int)min((int64_t)length, a.view.table_pitch << a.view.page_shift));
  return s;
}

// The pages that a wavefront is about to read, 64 of them a lane each, fetched when it comes to them.  (A page of 16 or more slots holds groups of 16 rows
// whole, so the page of a group is one number for the wavefront; smaller pages are looked up row by row.)
struct PageCursor {
  const int32_t* table;  // of the sequence
  int first, last;       // number of the first page held here; of the sequence's last one
  int32_t entry;
};
__device__ __forceinline__ int32_t checked_page(const PagedView& view, int32_t page) {
  if ((unsigned)page < (unsigned)view.pages) return page;
  page_error(view);
  return 0;
}
__device__ __forceinline__ void fetch_pages(const PagedView& view, PageCursor& at, int page) {
  at.first = page;
  at.entry = checked_page(view, at.table[min(page + (int)(threadIdx.x % kWave), at.last)]);
}
// Element of the cache at which the row of `key` begins; rows of a group of 16 follow each other.  For pages of 16 and more slots; key is uniform and a multiple
// of 16.
template <int D>
__device__ __forceinline__ int64_t group_offset(const PagedView& view, PageCursor& at, int kv_head, int key) {
  const int page = min(key >> view.page_shift, at.last);
  if (page - at.first >= kWave || page < at.first) fetch_pages(view, at, page);
  const int32_t entry = __builtin_amdgcn_readlane(at.entry, page - at.first);
  return ((((int64_t)entry * view.kv_heads + kv_head) << view.page_shift) + (key & ((1 << view.page_shift) - 1))) * D;
}
template <int D>
__device__ __forceinline__ int64_t row_offset(const PagedView& view, const PageCursor& at, int kv_head, int key) {
  const int32_t entry = checked_page(view, at.table[min(key >> view.page_shift, at.last)]);
  return ((((int64_t)entry * view.kv_heads + kv_head) << view.page_shift) + (key & ((1 << view.page_shift) - 1))) * D;
}

// 16-byte pieces of values: whether one holds an infinity or a NaN, and with those as zeros.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(const u32x4& x) {
  uint32_t found = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 4) found |= (x[w] & 0x7f800000u) == 0x7f800000u;
    else {
      constexpr uint32_t kExp = std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
      found |= (x[w] & kExp) == kExp || (x[w] & (kExp << 16)) == (kExp << 16);
    }
  }
  return found;
}
template <typename T>
__device__ __forceinline__ u32x4 finite_part(u32x4 x) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 4) x[w] = (x[w] & 0x7f800000u) == 0x7f800000u ? 0u : x[w];
    else {
      constexpr uint32_t kExp = std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
      if ((x[w] & kExp) == kExp) x[w] &= 0xffff0000u;
      if ((x[w] & (kExp << 16)) == (kExp << 16)) x[w] &= 0x0000ffffu;
    }
  }
  return x;
}

// What this lane gets of a 4 x 16 block of 16-bit values in LDS that lies row by row: four lanes point at the 32 bytes of a row, lane i of the sixteen gets column i.
__device__ __forceinline__ u32x2 read_transposed(const void* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
#else
  return u32x2{};
#endif
}

int launch_few_rows(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream);
int launch_tiles(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream);

}  // namespace ttmi
