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
  int every;  // this kernel takes all sequences: the other one is not launched
  // Of the few-rows kernel.  splits: how many workgroups share the work, 0: one for each sequence and key/value head; waves: of a workgroup; few: the rows of a sequence
  // that is its own (at most kFewRows).
  // Of the other.  Keys are cut at multiples of `chunk` (a multiple of 64), counted from the first of the sequence, so that no row sees more than `splits` parts (the
  // grid): a sequence that has more keys than was said takes longer ones.  Part p is in place p % splits.
  // ordered: its workgroups begin with those that have the most keys.
  int splits, waves, few, chunk, ordered;
  float* partial;  // sums of rows whose keys are several workgroups' [..][d], behind them the maxima and sums of their probabilities [..][2]
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
  // keys of a part (tiles).  A window's keys begin anywhere in a part, and so touch one more than they fill.
  __device__ __forceinline__ int chunk(const PagedArgs& a) const {
    if (a.splits <= 1) return INT32_MAX;
    const int seen = a.window > 0 ? min(length, a.window + tokens) : length, full = a.splits - (a.window > 0 ? 1 : 0);
    return max(a.chunk, ((seen + full - 1) / full + 63) & ~63);
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

// The pages that a wavefront is about to read, 64 of them, a lane each: where their rows of one key/value head begin; and the numbers of the 64 behind those, which are on
// their way.  A page of 16 or more slots holds groups of 16 rows whole, so where a group lies is one number for the wavefront (smaller pages are looked up row by row).
struct PageCursor {
  const int32_t* table;  // of the sequence
  int first, last;       // number of the first page held here; of the sequence's last one
  int32_t ahead;
  int64_t at;            // bytes
};
__device__ __forceinline__ int32_t checked_page(const PagedView& view, int32_t page) {
  if ((unsigned)page < (unsigned)view.pages) return page;
  page_error(view);
  return 0;
}
// Lanes past the sequence's last page hold that.
template <int ROW_BYTES>
__device__ __forceinline__ void hold_pages(const PagedView& view, PageCursor& c, int kv_head, int first, int32_t pages) {
  c.first = first;
  c.at = (((int64_t)checked_page(view, pages) * view.kv_heads + kv_head) << view.page_shift) * ROW_BYTES;
  c.ahead = c.table[min(first + kWave + (int)(threadIdx.x % kWave), c.last)];
}
template <int ROW_BYTES>
__device__ __forceinline__ void fetch_pages(const PagedView& view, PageCursor& c, int kv_head, int key) {
  const int page = key >> view.page_shift;
  hold_pages<ROW_BYTES>(view, c, kv_head, page, c.table[min(page + (int)(threadIdx.x % kWave), c.last)]);
}
// Before the groups of a tile are asked for.  (The 64 pages that are held end where a tile ends: tiles and their steps are powers of two, and so are pages.)
template <int ROW_BYTES>
__device__ __forceinline__ void come_to(const PagedView& view, PageCursor& c, int kv_head, int key) {
  const int past = (key >> view.page_shift) - c.first;
  if (__builtin_expect(past < kWave, 1)) return;
  if (past >= 2 * kWave) fetch_pages<ROW_BYTES>(view, c, kv_head, key);
  else hold_pages<ROW_BYTES>(view, c, kv_head, c.first + kWave, c.ahead);
}
// Byte of the cache at which the row of `key`, uniform and a multiple of 16, begins; the rows of its group follow.
template <int ROW_BYTES>
__device__ __forceinline__ int64_t group_at(const PagedView& view, const PageCursor& c, int key) {
  const int lane = (key >> view.page_shift) - c.first;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)c.at, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(c.at >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo) + (key & ((1 << view.page_shift) - 1)) * ROW_BYTES;
}
// Element at which any row begins, looked up.
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

// Both kernels are compiled as if there were no NaNs, which saves a canonicalising instruction for every operand of a maximum.  So what has to tell them asks for the bits of
// a number that was loaded as bits, and what adds one does it where the compiler does not look: it takes a test of a float for a test of infinity alone.
template <typename T>
using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
// sum += *at where that is an infinity or a NaN.  (Where its weight rounds to zero the matrix instruction, in tiles that all rows see, makes a NaN of an infinity: it multiplies.  Which of the
// two a token gets that sees one is not promised.)
template <typename T>
__device__ __forceinline__ void add_wild(float& sum, const T* at) {
  typedef Bits<T> __attribute__((may_alias)) Loaded;
  constexpr uint32_t kExp = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
  const uint32_t x = *reinterpret_cast<const Loaded*>(at);
  if ((x & kExp) != kExp) return;
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (std::is_same<T, f16>::value) {
    float wide;
    asm volatile("v_cvt_f32_f16 %1, %2\n\tv_add_f32 %0, %0, %1" : "+v"(sum), "=&v"(wide) : "v"(x));
  } else {
    asm volatile("v_add_f32 %0, %0, %1" : "+v"(sum) : "v"(sizeof(T) == 4 ? x : x << 16));
  }
#endif
}
// The reference point of a row's probabilities, in units of scale log2(e) score, a whole number: it moves only where a score lies more than this above it, so the sums are
// seldom scaled, and then by powers of two.  Probabilities of up to 2^8 lose no places: they are as exact in their type as those up to 1, and the division by their sum takes the factor back out.  What
// they cost is range: the sums before the division are at most 2^8 times the sum of |v| over the row's keys, which has to stay below 2^120 (fp16 values are far from that).  (The decision is the
// row's own: what is in the tile with it moves no bit of it.)
constexpr float kSlack = 8.f;
__device__ __forceinline__ float moved_reference(float top, float highest) { return highest > top + kSlack || top == -INFINITY ? fmaxf(__builtin_floorf(highest), top) : top; }

// What this lane gets of a 4 x 16 block of 16-bit values in LDS that lies row by row: four lanes point at the 32 bytes of a row, lane i of the sixteen gets column i.
__device__ __forceinline__ u32x2 read_transposed(const void* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
#else
  return u32x2{};
#endif
}

// What a row's sum is multiplied by in the end.  A row that sees no key has zeros.  Where one does, the sum of its probabilities is at least 1, or 0 if all its scores are
// minus infinity: then 0 times 1 / 0 makes the NaN that the division of zero by zero is.
__device__ __forceinline__ float inverse_sum(float sum, bool sees) { return sees ? 1.0f / sum : 0.f; }

// o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over `parts` partial results of a row, the p-th of which is row at(p) of `partial` [.., D] and `ml` [.., 2];
// sees: whether the row sees a key.  256 threads.
template <typename T, int D, typename At>
__device__ __forceinline__ void join_parts(const float* partial, const float* ml, int parts, bool sees, At at, T* out) {
  constexpr int kWide = 4, kThreads = D / kWide, kShares = 256 / kThreads;  // columns of a thread; threads of a part; parts at a time
  const int d0 = threadIdx.x % kThreads * kWide, share = threadIdx.x / kThreads;
  __shared__ float met[kShares][D + 2];
  // (each share with the maximum of its own parts)
  float best = -INFINITY;
  for (int p = share; p < parts; p += kShares) best = fmaxf(best, ml[2 * at(p)]);
  const float zero = best == -INFINITY ? 0.f : best;
  float total = 0.f;
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = share; p < parts; p += kShares) {
    const int64_t row = at(p);
    const float weight = __builtin_amdgcn_exp2f(ml[2 * row] - zero);
    total += ml[2 * row + 1] * weight;
    sum += *reinterpret_cast<const floatx4*>(partial + row * D + d0) * weight;
  }
#pragma unroll
  for (int c = 0; c < kWide; ++c) met[share][d0 + c] = sum[c];
  if (d0 == 0) met[share][D] = best, met[share][D + 1] = total;
  __syncthreads();
  if ((int)threadIdx.x >= D) return;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kShares; ++i) top = fmaxf(top, met[i][D]);
  const float base = top == -INFINITY ? 0.f : top;
  float l = 0.f, x = 0.f;
#pragma unroll
  for (int i = 0; i < kShares; ++i) {
    const float weight = __builtin_amdgcn_exp2f(met[i][D] - base);
    l += met[i][D + 1] * weight;
    x += met[i][threadIdx.x] * weight;
  }
  out[threadIdx.x] = from_float<T>(sees ? x / l : 0.f);
}

// The same for one wavefront and few parts: four columns a lane, the parts shared by the lanes that are left.
template <typename T, int D, typename At>
__device__ __forceinline__ void join_parts_by_wavefront(const float* partial, const float* ml, int parts, bool sees, At at, T* out) {
  constexpr int kThreads = D / 4, kShares = kWave / kThreads;
  const int lane = (int)(threadIdx.x % kWave), d0 = lane % kThreads * 4, share = lane / kThreads;
  float best = -INFINITY;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) best = fmaxf(best, ml[2 * at(p)]);
  const float zero = best == -INFINITY ? 0.f : best;
  float total = 0.f;
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = share; p < parts; p += kShares) {
    const int64_t row = at(p);
    const float weight = __builtin_amdgcn_exp2f(ml[2 * row] - zero);
    total += ml[2 * row + 1] * weight;
    sum += *reinterpret_cast<const floatx4*>(partial + row * D + d0) * weight;
  }
#pragma unroll
  for (int d = kThreads; d < kWave; d *= 2) {
    total += __shfl_xor(total, d, kWave);
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] += __shfl_xor(sum[c], d, kWave);
  }
  if (share != 0) return;
  const float inv = inverse_sum(total, sees);
  Vec<T, 4> x;
#pragma unroll
  for (int c = 0; c < 4; ++c) x.v[c] = from_float<T>(sum[c] * inv);
  store_vec<T, 4>(out + d0, x);
}

int launch_few_rows(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream);
int launch_tiles(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream);

}  // namespace ttmi
