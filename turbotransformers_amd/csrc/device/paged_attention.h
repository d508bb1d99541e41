// What the kernels of attention over pages share: their arguments, which keys a row sees and which part of them is whose, where rows of the cache lie.
//
// The rows of one sequence and key/value head are its new tokens' query heads of that group, token by token: row r is head r % group of the group, token
// r / group, so a tile of rows reads each key and value once for all heads that share it.
#pragma once

#include "attention_common.h"
#include "paged.h"

namespace ttmi {

constexpr int kFewRows = 16;  // rows of a sequence and key/value head that are the few-rows kernel's
constexpr int kShareStep = 128;  // keys of a family are taken in steps of this, a multiple of every tile: what is left of them is each sequence's own

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
  // Of the kernels that know of first keys that stay visible and of families (SIGHT).
  int sinks;
  const int32_t* families;  // null: none
  // shares: workgroups that the families' keys, in at most family_splits parts of at least family_least steps of 64, and the sequences with few rows take among them;
  // few_splits, few_every: splits and every of the few-rows kernel, where it runs (run_few); own_blocks: blocks of 128 rows of sequences' own keys, tile_groups workgroups.
  // family_few: rows of a family up to which it is the few-rows kernel's, in blocks of kFewRows, where that is among those workgroups.
  int shares, family_splits, family_least, family_few, run_few, few_splits, few_every, own_blocks, tile_groups;
  // With families `partial` holds the rows of all results that are joined: those of the few-rows kernel (2 splits kFewRows), and from these on, for each row of q and head:
  int64_t own_at, family_at, whole_at, rows;  // of a sequence's own keys in parts, of its family's in parts, of its own where one workgroup had them all; the end
};

struct Reach {
  int begin, end;  // keys
  int low;         // SIGHT: keys below, from the sequence's own first on, are seen besides
};
struct Sequence {
  int start, tokens, length, first;  // its first row, new tokens, keys, position of the first new token
  int base = 0;                      // SIGHT: keys below are its family's
  __device__ __forceinline__ Reach reach(const PagedArgs& a, int token) const {
    const int position = first + token;
    Reach r;
    r.begin = a.window > 0 ? max(0, position - a.window + 1) : 0;
    r.end = a.causal ? max(0, min(length, position + 1)) : length;
    if (r.begin >= r.end) r.begin = r.end = 0;
    r.low = 0;
    return r;
  }
  // The same with the first keys that stay visible, of the sequence's own keys alone (where it sees none of them, begin, end and low are `base`); all ends rise with the token.
  __device__ __forceinline__ Reach own_reach(const PagedArgs& a, int token) const {
    Reach r = reach(a, token);
    r.low = max(base, a.window > 0 ? min(a.sinks, r.end) : 0);
    r.end = max(base, r.end);
    r.begin = min(max(base, r.begin), r.end);
    return r;
  }
  template <bool SIGHT>
  __device__ __forceinline__ Reach reach_of(const PagedArgs& a, int token) const {
    if constexpr (SIGHT) return own_reach(a, token);
    else return reach(a, token);
  }
  // keys of a part (tiles).  A window's keys begin anywhere in a part, and so touch one more than they fill.
  __device__ __forceinline__ int chunk(const PagedArgs& a) const {
    if (a.splits <= 1) return INT32_MAX;
    const int seen = a.window > 0 ? min(length, a.window + tokens) : length, full = a.splits - (a.window > 0 ? 1 : 0);
    return max(a.chunk, ((seen + full - 1) / full + 63) & ~63);
  }
  // SIGHT: the same of the keys that a block of its rows sees, laid behind each other (Span): whole tiles of first keys, a window that begins anywhere in a tile.
  __device__ __forceinline__ int span_chunk(const PagedArgs& a) const {
    if (a.splits <= 1) return INT32_MAX;
    const int own = max(0, length - base);
    const int seen = a.window > 0 ? (int)min((int64_t)own, (int64_t)max(0, a.sinks - base) + a.window + tokens + 128) : own;
    return max(a.chunk, ((seen + a.splits - 1) / a.splits + 63) & ~63);
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

// Keys that a block of rows sees: those from first to end, of which all rows see those from sure_first to sure_end; SIGHT: and those below low, of which all see those below
// sure_low.
struct Sight {
  int first, end, sure_first, sure_end, low, sure_low;
};
// Of rows whose ends rise from the first to the last.  (A row without keys, before the first one that has some, begins and ends where the sequence's own keys do.)
__device__ __forceinline__ Sight sight_of(const Reach& first_row, const Reach& last_row) {
  Sight s;
  s.first = first_row.begin, s.end = max(first_row.end, last_row.end), s.sure_first = last_row.begin, s.sure_end = first_row.end;
  s.low = max(first_row.low, last_row.low), s.sure_low = min(first_row.low, last_row.low);
  return s;
}
template <bool SIGHT>
__device__ __forceinline__ bool all_see(const Sight& s, int key, int keys) {
  return (key >= s.sure_first && key + keys <= s.sure_end) || (SIGHT && key + keys <= s.sure_low);
}
template <bool SIGHT>
__device__ __forceinline__ bool some_see(const Sight& s, int key) {
  return (key >= s.first && key < s.end) || (SIGHT && key < s.low);
}
template <bool SIGHT>
__device__ __forceinline__ bool sees(const Reach& r, int key) {
  return (key >= r.begin && key < r.end) || (SIGHT && key < r.low);
}
// SIGHT: whole tiles of the first keys that some row sees and, right behind them, whole tiles of the others: places lo to hi, the tile at a place holds the keys from key_at on.
struct Span {
  int lo, hi, seam, skip;
  __device__ __forceinline__ int key_at(int place) const { return place + (place >= seam ? skip : 0); }
  __device__ __forceinline__ int place_of(int key) const { return key - (key >= seam + skip ? skip : 0); }
};
template <int TILE>
__device__ __forceinline__ Span span_of(const Sight& s, int base) {
  Span span;
  const int start = s.first & ~(TILE - 1);
  if (s.low <= base) return {start, s.end, 0, 0};
  span.seam = (s.low + TILE - 1) & ~(TILE - 1);
  span.skip = max(0, start - span.seam);
  span.lo = base, span.hi = s.end - span.skip;
  return span;
}

// Sums over the lanes up to this one, it included, and over all.
__device__ __forceinline__ int sum_up_to_here(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}
__device__ __forceinline__ int sum_of_lanes(int v) { return __builtin_amdgcn_readlane(sum_up_to_here(v), kWave - 1); }

// A family: sequences that follow one another and begin with the same keys.  A sequence is of a family where its row of `families` is, number by number, that of the first sequence that it
// names: any other is on its own, whatever either says, so that no key is left out, read twice or taken from another text.  Decided in lane_sequences and, for rows of sequences that are
// not among the 64 at hand, in family_reach.
struct Family {
  int first, end, keys;  // sequences; keys in common, a multiple of kShareStep, 0: no family
};
// Keys that a sequence whose row is `row` has in common with the first one that it names, which is before the 64 at hand.
__device__ __forceinline__ int keys_in_common(const PagedArgs& a, const int (&row)[3]) {
  const PagedView& view = a.view;
  const int32_t* const its = a.families + 3 * (int64_t)row[0];
  const int held = (int)min((int64_t)view.lengths[row[0]], view.table_pitch << view.page_shift);
  return its[0] == row[0] && its[1] == row[1] && its[2] == row[2] ? max(0, min(row[2], held)) & ~(kShareStep - 1) : 0;
}

// 64 sequences, a lane each, with one trip to memory: what they are, the families that they lead and whose keys are not their own.
struct LaneSequences {
  int base;                            // number of the first
  int starts, ends;                    // of the packed rows, as they are given
  int start, tokens, length, first, own;  // as in Sequence (own: its base)
  int leader;                          // the first of its family; -1: it is on its own
  int family_end, family_keys, family_tokens;  // of the family that it leads; keys 0: none

  __device__ __forceinline__ Sequence sequence(int lane) const {
    Sequence s;
    s.start = __builtin_amdgcn_readlane(start, lane), s.tokens = __builtin_amdgcn_readlane(tokens, lane), s.length = __builtin_amdgcn_readlane(length, lane);
    s.first = __builtin_amdgcn_readlane(first, lane), s.base = __builtin_amdgcn_readlane(own, lane);
    return s;
  }
  __device__ __forceinline__ Family family(int lane) const {
    return {base + lane, __builtin_amdgcn_readlane(family_end, lane), __builtin_amdgcn_readlane(family_keys, lane)};
  }
  // A family as a sequence: the rows of all of its sequences over the keys they have in common.
  __device__ __forceinline__ Sequence family_sequence(int lane) const {
    Sequence s;
    s.start = __builtin_amdgcn_readlane(start, lane), s.tokens = __builtin_amdgcn_readlane(family_tokens, lane);
    s.length = __builtin_amdgcn_readlane(family_keys, lane), s.first = 0;
    return s;
  }
};
struct LaneNumbers {  // as they are given
  int starts, ends, length, row[3];
};
__device__ __forceinline__ LaneNumbers lane_numbers(const PagedArgs& a, int base) {
  const int at = min(base + (int)(threadIdx.x % kWave), a.view.batch - 1);
  LaneNumbers n = {a.view.starts[at], a.view.starts[at + 1], a.view.lengths[at], {-1, 0, 0}};
  if (a.families != nullptr) {
#pragma unroll
    for (int i = 0; i < 3; ++i) n.row[i] = a.families[3 * (int64_t)at + i];
  }
  return n;
}
__device__ __forceinline__ LaneSequences lane_sequences(const PagedArgs& a, int base, const LaneNumbers& numbers) {
  const PagedView& view = a.view;
  const int lane = (int)(threadIdx.x % kWave), b = base + lane;
  LaneSequences s;
  s.base = base;
  s.starts = numbers.starts, s.ends = numbers.ends;
  const int length = numbers.length;
  const int(&row)[3] = numbers.row;
  const int held = (int)min((int64_t)length, view.table_pitch << view.page_shift);
  s.start = max(0, s.starts), s.tokens = b < view.batch ? max(0, min(s.ends, view.tokens) - s.start) : 0;
  s.length = max(0, held), s.first = length - s.tokens;
  s.own = 0, s.leader = -1, s.family_end = min(row[1], view.batch), s.family_keys = s.family_tokens = 0;
  if (a.families == nullptr) return s;
  if (b < view.batch && row[0] == b && s.family_end > b + 1) s.family_keys = max(0, min(row[2], held)) & ~(kShareStep - 1);
  const int last = s.family_end - 1 - base;
  int rows_end = __shfl(s.ends, max(0, min(last, kWave - 1)), kWave);
  if (s.family_keys > 0 && last >= kWave) rows_end = view.starts[s.family_end];
  if (s.family_keys > 0) s.family_tokens = max(0, min(rows_end, view.tokens) - s.start);
  const int from = row[0] - base, there = max(0, min(from, kWave - 1));
  int keys = __shfl(s.family_keys, there, kWave);
  const int its_end = __shfl(row[1], there, kWave), its_keys = __shfl(row[2], there, kWave);
  if (its_end != row[1] || its_keys != row[2] || b >= s.family_end) keys = 0;
  if ((unsigned)row[0] > (unsigned)b) keys = 0;
  else if (from < 0) keys = b < s.family_end ? keys_in_common(a, row) : 0;
  if (keys > 0) s.own = keys, s.leader = row[0];
  return s;
}
__device__ __forceinline__ LaneSequences lane_sequences(const PagedArgs& a, int base) { return lane_sequences(a, base, lane_numbers(a, base)); }
// Blocks of kFewRows rows of a lane's family, where the few-rows kernel takes it, and its rows of 128, where that of many rows does.
struct FamilyBlocks {
  int few, many;
};
__device__ __forceinline__ FamilyBlocks family_blocks(const PagedArgs& a, const LaneSequences& lanes) {
  const int64_t rows = (int64_t)lanes.family_tokens * a.group;
  const bool few = rows <= a.family_few;
  return {few ? (int)(rows + kFewRows - 1) / kFewRows : 0, few ? 0 : (int)((rows + 127) / 128)};
}
// The keys of a part that some row of a family's block sees: from lo to hi, shortened (both stay multiples of TILE, or the end of what is seen).  With a window these are the first keys that stay
// visible, the windows' or, from the one to the other, both.
template <int TILE>
__device__ __forceinline__ void seen_of_part(const Sight& s, int* lo, int* hi) {
  if (*lo >= s.low) *lo = max(*lo, min(*hi, s.first & ~(TILE - 1)));
  *hi = min(*hi, s.end);
  if (*hi <= s.first) *hi = min(*hi, s.low);
  *hi = max(*lo, *hi);
}
// The sequence of a family that a row of q belongs to, each lane's own, and what of the family's keys the row sees; *member: whether that sequence is of the family.  Where each
// sequence has one new token and they lie among the 64, no trip to memory.
__device__ __forceinline__ Reach family_reach(const PagedArgs& a, const LaneSequences& s, const Family& f, int start, int row, bool* member) {
  const PagedView& view = a.view;
  const int guess = min(f.first + row - start, f.end - 1), at = min(guess - s.base, kWave - 1);
  *member = __shfl(s.leader, at, kWave) == f.first;
  Sequence q;
  q.start = __shfl(s.start, at, kWave), q.tokens = __shfl(s.tokens, at, kWave), q.length = __shfl(s.length, at, kWave), q.first = __shfl(s.first, at, kWave);
  if (!(guess - s.base < kWave && q.start <= row && row < q.start + q.tokens)) {
    int lo = f.first, hi = f.end;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (view.starts[mid] <= row) lo = mid;
      else hi = mid;
    }
    q = sequence(a, lo);
    const int32_t *const its = a.families + 3 * (int64_t)lo, *const firsts = a.families + 3 * (int64_t)f.first;
    *member = its[0] == f.first && its[1] == firsts[1] && its[2] == firsts[2];
  }
  Reach r = q.reach(a, row - q.start);
  r.low = min(f.keys, a.window > 0 ? min(a.sinks, r.end) : 0);
  r.end = min(f.keys, r.end);
  r.begin = min(r.begin, r.end);
  return r;
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
// SIGHT: behind a gap lie pages that are known from the start, so their numbers are asked for with the first ones and not when the gap is reached (which costs a workgroup a trip to memory).
struct GapCursor : PageCursor {
  int next;  // number of the first page that `ahead` is of
};
template <int ROW_BYTES>
__device__ __forceinline__ void fetch_pages(const PagedView& view, GapCursor& c, int kv_head, int key, int behind) {
  fetch_pages<ROW_BYTES>(view, c, kv_head, key);
  c.next = c.first + kWave;
  if (behind > key) {
    c.next = behind >> view.page_shift;
    c.ahead = c.table[min(c.next + (int)(threadIdx.x % kWave), c.last)];
  }
}
template <int ROW_BYTES>
__device__ __forceinline__ void come_to(const PagedView& view, GapCursor& c, int kv_head, int key) {
  const int page = key >> view.page_shift;
  if (__builtin_expect(page - c.first < kWave, 1)) return;
  if ((unsigned)(page - c.next) < (unsigned)kWave) hold_pages<ROW_BYTES>(view, c, kv_head, c.next, c.ahead);
  else fetch_pages<ROW_BYTES>(view, static_cast<PageCursor&>(c), kv_head, key);
  c.next = c.first + kWave;
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

// How the work of a call is laid out: `all` for the launch of everything, `few` for that of the sequences with few rows where they have one of their own.
struct SightLaunch {
  PagedArgs all, few;
  bool run_tiles;
};
void launch_sight_f16(const SightLaunch& l, int64_t head_dim, hipStream_t stream);
void launch_sight_bf16(const SightLaunch& l, int64_t head_dim, hipStream_t stream);
void launch_sight_f32(const SightLaunch& l, int64_t head_dim, hipStream_t stream);

}  // namespace ttmi
