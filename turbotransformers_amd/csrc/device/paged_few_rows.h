// Attention over pages where a sequence has few rows (new tokens times query heads of a key/value head): decoding.
//
// What it has to read, every key and value once, bounds it.  A workgroup has up to 16 rows of one sequence and head and a part of the keys; its NW wavefronts (four,
// or eight where a launch leaves CUs without a workgroup) take its tiles in turn, each with a running maximum, sum and output of its own, without a barrier until they meet at the end.  Scores are
// computed transposed,
//     St[key, row] = K[key, :] . Q[row, :]        v_mfma_f32_16x16x32 (fp32: 16x16x4), K as it comes from memory, a 16-byte piece of a row a lane,
// so a lane has one row and four keys of each 16: the statistics need one exchange over the four quarters of the wavefront, and the probabilities lie as the
// second operand of
//     Ot[d, row] += Vt[d, keys] . Pt[keys, row]
// wants them: its order of keys is ours to choose.  Vt is what the transposing reads give of a tile that lies in LDS row by row as it came (fp32: plain reads of a
// column).  Tiles are fetched into registers one ahead: 8 KB of keys and as many of values per wavefront are on their way while one is worked on; what a CU has on its way is
// what it gets (about 50 GB/s while the others leave the memory room for that; 20 where all 256 read, which is its 5 TB/s), so the loads are never behind a condition, which would make
// the compiler wait for all of them.
//
// Measured, 32 query and 8 key heads of 128: 64 sequences of 100 to 6000 keys, bf16, 85 us and 6 to join the parts (5.1 TB/s while it reads; a large copy here 4.8);
// 4 sequences of 60000 to 131071 keys, fp16, 264 and 7 (6.0 TB/s, part of it out of the last-level cache).  One sequence of 387 keys, 12 heads of 64, fp16: 6.7, of which
// most is the trips to memory that follow one another: length, pages, keys.
//
// kSinks, kFamilies: rows that see the first keys of their sequence besides a window, and sequences whose first keys are their family's (another kernel's).  The keys that a pair's rows see are laid
// behind each other in whole tiles (Span), so that rounds and tiles go over them without the gap.
#pragma once

#include "paged_attention.h"

namespace ttmi {
namespace {

template <typename T, int D, int NW>
struct FewRows {
  static constexpr int kKeys = sizeof(T) == 2 ? 32 : 16;        // of a tile
  static constexpr int kElems = 16 / (int)sizeof(T);            // of a 16-byte piece
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kSteps = kRowBytes / 64;                 // pieces of a row per lane
  static constexpr int kGroups = kKeys / 16;
  static constexpr int kValuePieces = 16 * kRowBytes / 1024;    // per lane and group
  static constexpr int kTiles = D / 16;                         // of the output
  static constexpr int kValueBytes = kKeys * kRowBytes;         // of a wavefront, in LDS
  static constexpr int kPitch = D + 4;                          // floats of a row where the wavefronts meet
  static constexpr int kMergeBytes = NW * kFewRows * kPitch * 4;
  static constexpr int kLds = NW * kValueBytes > kMergeBytes ? NW * kValueBytes : kMergeBytes;
};

// Place of a 16-byte piece in a row of a tile of values: the transposing reads take 32 bytes of each of sixteen rows at a time, plain ones 64 bytes of four rows
// that lie four apart, and both find them in different banks so.
template <typename T, int D>
__device__ __forceinline__ int value_piece(int row, int piece) {
  if constexpr (sizeof(T) == 4) return piece ^ (((row >> 2) & 3) << 2);
  else if constexpr (D == 128) return piece ^ ((row & 7) << 1);
  else return piece ^ (((row >> 1) & 3) << 1);
}

template <typename T>
__device__ __forceinline__ floatx4 mma16(const u32x4& a, const u32x4& b, floatx4 c) {
  if constexpr (std::is_same<T, f16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
  else if constexpr (std::is_same<T, bf16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else {
    const floatx4 x = __builtin_bit_cast(floatx4, a), y = __builtin_bit_cast(floatx4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
}

// Over the four quarters of the wavefront, which hold the same row.
__device__ __forceinline__ float quarters_max(float v) {
  LanePair p = swap_rows(v);
  v = fmaxf(p.a, p.b);
  p = swap_halves(v);
  return fmaxf(p.a, p.b);
}
__device__ __forceinline__ float quarters_sum(float v) {
  LanePair p = swap_rows(v);
  v = p.a + p.b;
  p = swap_halves(v);
  return p.a + p.b;
}

// The work is cut evenly over the workgroups whatever the sequences' lengths: a unit is a round, kRound keys of one sequence and key/value head, units are counted
// sequence by sequence, head by head, and workgroup w of W takes those from w R / W to (w + 1) R / W.  So of the pairs of a sequence and a head that it meets only the first
// and the last can be another's too; their partial results have a place each.
constexpr int kRound = 128;
// A pair has a unit more than rounds: what a workgroup waits for when it comes to one (its length, its pages, its first tile) is time that others have for theirs.
// us, 64 sequences of 100 to 6000 keys (three draws, and all of 1450), without / with it / with two: 105 / 89 / 91, 87 / 75 / 77, 107 / 94 / 97, 104 / 95 / 98, 75 / 75 / 75.
constexpr int kStart = 1;
// Of this lane (without tokens behind the last sequence).
__device__ __forceinline__ Sequence own_sequence(const LaneSequences& lanes) {
  Sequence s;
  s.start = lanes.start, s.tokens = lanes.tokens, s.length = lanes.length, s.first = lanes.first, s.base = lanes.own;
  return s;
}
constexpr int kWindow = 0, kSinks = 1, kFamilies = 2;  // what a kernel knows of: windows alone; first keys that stay visible; families, too
struct Walk {  // 64 sequences, a lane each
  LaneSequences lanes;    // kFamilies
  int base, rounds;       // number of the first; rounds of this lane's, for one head
  int family_rounds, family_blocks;  // kFamilies: the same of the family that it leads, for one head and block of rows, and those blocks: they come first
  int64_t before, upto;   // units of all sequences before these; of these up to this lane's, it included
  int64_t groups;         // of batches of more than 64 sequences: units of this lane's 64th of them and of those before it (kFamilies: or `ahead`: not counted, the walk only goes on)
  bool ahead;
};
constexpr int kSpanTile = 32;  // a tile or two
template <bool SIGHT>
__device__ __forceinline__ int rounds_of(const PagedArgs& a, const Sequence& seq) {
  const int rows = seq.tokens * a.group;
  if (rows <= 0) return 0;
  if (rows > a.few) return (SIGHT ? a.few_every : a.every) ? kStart + 1 : 0;  // (more rows than was said: not cut)
  if constexpr (SIGHT) {
    const Span span = span_of<kSpanTile>(sight_of(seq.own_reach(a, 0), seq.own_reach(a, seq.tokens - 1)), seq.base);
    return kStart + max(1, (span.hi - span.lo + kRound - 1) / kRound);
  }
  const Reach low = seq.reach(a, 0), high = seq.reach(a, seq.tokens - 1);
  return kStart + max(1, (max(low.end, high.end) + kRound - 1) / kRound - low.begin / kRound);
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t sum_up_to_lane(int64_t v) {
  const int lane = (int)(threadIdx.x % kWave);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t below = __shfl_up((long long)v, d, kWave);
    if (lane >= d) v += below;
  }
  return v;
}
// Rounds of a lane's family, for one head and block of kFewRows rows (0: none here), and of all there are for one head.
__device__ __forceinline__ int family_rounds_of(const LaneSequences& lanes, int blocks) { return blocks > 0 ? kStart + lanes.family_keys / kRound : 0; }
__device__ __forceinline__ int all_rounds_of(const PagedArgs& a, const LaneSequences& lanes) {
  const int blocks = a.families != nullptr ? family_blocks(a, lanes).few : 0;
  return rounds_of<true>(a, own_sequence(lanes)) + blocks * family_rounds_of(lanes, blocks);
}
__device__ __forceinline__ void take_lanes(const PagedArgs& a, Walk& w) {
  w.rounds = rounds_of<true>(a, own_sequence(w.lanes));
  w.family_blocks = a.families != nullptr ? family_blocks(a, w.lanes).few : 0, w.family_rounds = family_rounds_of(w.lanes, w.family_blocks);
  w.upto = (int64_t)sum_up_to_here(w.rounds + w.family_blocks * w.family_rounds) * a.view.kv_heads;
}
template <int SEES>
__device__ __forceinline__ void walk_to(const PagedArgs& a, Walk& w, int base, int64_t before) {
  w.base = base, w.before = before;
  if constexpr (SEES == kFamilies) {
    w.lanes = lane_sequences(a, base);
    take_lanes(a, w);
  } else {
    const int lane = (int)(threadIdx.x % kWave);
    w.rounds = base + lane < a.view.batch ? rounds_of<SEES == kSinks>(a, sequence(a, base + lane)) : 0;
    w.upto = sum_up_to_lane((int64_t)w.rounds * a.view.kv_heads);
  }
}
template <int SEES>
__device__ __forceinline__ void walk_on(const PagedArgs& a, Walk& w) { walk_to<SEES>(a, w, w.base + kWave, w.before + lane_of(w.upto, kWave - 1)); }
__device__ __forceinline__ int group_size(const PagedArgs& a) { return (a.view.batch + kWave - 1) / kWave; }
template <int SEES>
__device__ __forceinline__ void walk_to_group(const PagedArgs& a, Walk& w, int group) {
  walk_to<SEES>(a, w, group * group_size(a), group > 0 ? lane_of(w.groups, group - 1) : 0);
}
// -> all units
template <int SEES>
__device__ __forceinline__ int64_t count_units(const PagedArgs& a, Walk& w) {
  w.groups = 0;
  if (a.view.batch <= kWave) {
    walk_to<SEES>(a, w, 0, 0);
    return lane_of(w.upto, kWave - 1);
  }
  const int size = group_size(a), first = (int)(threadIdx.x % kWave) * size;
  int64_t mine = 0;
  if constexpr (SEES == kFamilies) {
    // 64 sequences at a time; what each group of `size` has is kept by its lane
    for (int base = 0; base < a.view.batch; base += kWave) {
      const int upto = sum_up_to_here(all_rounds_of(a, lane_sequences(a, base)));
      const int from = min(max(first - base, 0), kWave), to = min(max(first + size - base, 0), kWave);
      const int low = __shfl(upto, max(from - 1, 0), kWave), high = __shfl(upto, max(to - 1, 0), kWave);
      mine += (to > 0 ? high : 0) - (from > 0 ? low : 0);
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < size; ++i) mine += first + i < a.view.batch ? rounds_of<SEES == kSinks>(a, sequence(a, first + i)) : 0;
  }
  w.groups = sum_up_to_lane(mine * a.view.kv_heads);
  w.base = 0, w.rounds = 0, w.before = w.upto = 0;
  return lane_of(w.groups, kWave - 1);
}
struct Place {
  int b, kv_head, round, rounds;  // round: of this head's `rounds`
  int block = -1;                 // kFamilies: of the rows of the family that b leads
};
template <int SEES>
__device__ __forceinline__ Place find_unit(const PagedArgs& a, Walk& w, int64_t unit) {
  if (a.view.batch > kWave && !(SEES == kFamilies && w.ahead) && (unit < w.before || unit >= w.before + lane_of(w.upto, kWave - 1)))
    walk_to_group<SEES>(a, w, __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(w.groups > unit)) - 1));
  while (w.before + lane_of(w.upto, kWave - 1) <= unit) walk_on<SEES>(a, w);
  const int64_t at = unit - w.before;
  const int found = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(w.upto > at)) - 1);
  Place p;
  p.b = w.base + found, p.rounds = __builtin_amdgcn_readlane(w.rounds, found);
  if constexpr (SEES == kFamilies) {
    const int blocks = __builtin_amdgcn_readlane(w.family_blocks, found), family_rounds = __builtin_amdgcn_readlane(w.family_rounds, found);
    int rest = (int)(at - (lane_of(w.upto, found) - (int64_t)(p.rounds + blocks * family_rounds) * a.view.kv_heads));
    const int of_family = blocks * family_rounds * a.view.kv_heads;
    if (rest < of_family) {
      p.rounds = family_rounds;
      const int pair = rest / family_rounds;
      p.round = rest - pair * family_rounds, p.block = pair / a.view.kv_heads, p.kv_head = pair - p.block * a.view.kv_heads;
    } else {
      rest -= of_family;
      p.kv_head = rest / p.rounds, p.round = rest - p.kv_head * p.rounds;
    }
  } else {
    const int rest = (int)(at - (lane_of(w.upto, found) - (int64_t)p.rounds * a.view.kv_heads));
    p.kv_head = rest / p.rounds, p.round = rest - p.kv_head * p.rounds;
  }
  return p;
}
// a / b of numbers that are not negative: a division of 64 bits takes longer than a trip to L2, and they are seldom needed.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (__builtin_expect((((uint64_t)a | (uint64_t)b) >> 32) == 0, 1)) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
// Workgroups that share the work.  At least kFewest rounds each, so that a wavefront has more than its first tile's wait.  us, 1 / 2 / 4 of them, 8 key heads of 128: 1 sequence
// of 1500 keys 11.6 / 12.5 / 15.6, of 8000 16.4 / 14.1 / 15.6, 8 of 1000 19.0 / 16.7 / 17.7, 8 of 2000 21.2 / 21.4 / 25.8.
constexpr int kFewest = 2;
__device__ __forceinline__ int64_t sharers(int splits, int64_t units) { return max((int64_t)1, min((int64_t)splits, (units + kFewest - 1) / kFewest)); }

template <typename T, int D, int NW>
struct FewRowsShared {
  __align__(16) char tiles[FewRows<T, D, NW>::kLds];
  float met[NW][kFewRows][2];
  int theirs[kFewRows];  // kFamilies: of a family's rows, whether they are
};

// The share of one of `splits` workgroups (0: of a pair); kFamilies: units and walk as count_units gives them, if units >= 0.  SMALL: pages of fewer than 16 slots
template <typename T, int D, int NW, bool SMALL, int SEES>
__device__ __forceinline__ void few_rows(const PagedArgs& a, int workgroup, int splits, Walk& walk, int64_t all_units, FewRowsShared<T, D, NW>& shared) {
  using S = FewRows<T, D, NW>;
  constexpr bool SIGHT = SEES != kWindow, FAMILIES = SEES == kFamilies;
  char* const smem = shared.tiles;
  auto& met = shared.met;
  const PagedView& view = a.view;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = lane & 15, quarter = lane >> 4;
  const T* const q = static_cast<const T*>(a.q);
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  char* const tile = smem + wave * S::kValueBytes;

  // splits 0: a workgroup for each pair
  int64_t unit = workgroup, stop = unit + 1;
  if (splits > 0) {
    const int64_t units = FAMILIES && all_units >= 0 ? all_units : count_units<SEES>(a, walk), workgroups = sharers(splits, units);
    if (workgroup >= workgroups) return;
    if constexpr (SIGHT) unit = quotient(units * workgroup, workgroups), stop = quotient(units * (workgroup + 1), workgroups);
    else unit = units * workgroup / workgroups, stop = units * (workgroup + 1) / workgroups;
  }
  while (unit < stop) {
    Place place;
    if (splits > 0) place = find_unit<SEES>(a, walk, unit);
    else place.b = (int)(unit / view.kv_heads), place.kv_head = (int)(unit % view.kv_heads), place.round = 0, place.rounds = INT32_MAX;
    const int b = place.b, kv_head = place.kv_head;
    const int64_t ends = splits > 0 ? min(stop, unit + place.rounds - place.round) : stop;
    const int start = splits > 0 ? kStart : 0;  // (in a pair's first unit there is nothing to do)
    const int round0 = max(0, place.round - start), round1 = place.round + (int)(splits > 0 ? ends - unit : INT32_MAX) - start;
    const bool complete = round0 == 0 && round1 == place.rounds - start;
    unit = ends;
    if (round1 <= round0) continue;
    Sequence seq;
    Family family{};
    if constexpr (FAMILIES) {
      if (splits == 0) walk.lanes = lane_sequences(a, b & ~(kWave - 1));
      seq = walk.lanes.sequence(b - walk.lanes.base);
      if (place.block >= 0) family = walk.lanes.family(b - walk.lanes.base), seq = walk.lanes.family_sequence(b - walk.lanes.base);
    } else seq = sequence(a, b);
    const bool of_family = FAMILIES && place.block >= 0;
    const int rows_all = of_family ? min(seq.tokens * a.group, (place.block + 1) * kFewRows) : seq.tokens * a.group;
    if (!of_family && (rows_all <= 0 || (rows_all > a.few && !(SIGHT ? a.few_every : a.every)))) return;  // (a workgroup of its own)
    if (round0 == 0 && kv_head == 0 && tid == 0 && !of_family && view.lengths[b] > seq.length) page_error(view);
    typename std::conditional<SIGHT, GapCursor, PageCursor>::type cursor;
    cursor.table = view.table + (int64_t)b * view.table_pitch;
    cursor.first = 0, cursor.ahead = 0, cursor.at = 0;

    for (int row0 = of_family ? place.block * kFewRows : 0; row0 < rows_all; row0 += kFewRows) {
      const int rows = min(kFewRows, rows_all - row0);
      const int token0 = row0 / a.group, token1 = (row0 + rows - 1) / a.group;
      const int token = row < rows ? (row0 + row) / a.group : token0, head = kv_head * a.group + (row < rows ? row0 + row - token * a.group : 0);
      Reach mine;
      Sight sight;
      Span span;
      int lo, hi;  // SIGHT: places
      if (of_family) {
        bool member;
        mine = family_reach(a, walk.lanes, family, seq.start, seq.start + token, &member);
        if (wave == 0 && quarter == 0) shared.theirs[row] = member;
        sight = {0, family.keys, 0, family.keys, 0, 0};
        if (!__all(mine.begin == 0 && mine.end == family.keys && mine.low == 0)) {  // (lanes without a row have the first one's)
          sight = {mine.begin, mine.end, mine.begin, mine.end, mine.low, mine.low};
#pragma unroll 1
          for (int d = 1; d < kFewRows; d *= 2) {
            sight.first = min(sight.first, __shfl_xor(sight.first, d, kWave)), sight.end = max(sight.end, __shfl_xor(sight.end, d, kWave));
            sight.sure_first = max(sight.sure_first, __shfl_xor(sight.sure_first, d, kWave)), sight.sure_end = min(sight.sure_end, __shfl_xor(sight.sure_end, d, kWave));
            sight.low = max(sight.low, __shfl_xor(sight.low, d, kWave)), sight.sure_low = min(sight.sure_low, __shfl_xor(sight.sure_low, d, kWave));
          }
          sight = {__builtin_amdgcn_readfirstlane(sight.first), __builtin_amdgcn_readfirstlane(sight.end), __builtin_amdgcn_readfirstlane(sight.sure_first),
                   __builtin_amdgcn_readfirstlane(sight.sure_end), __builtin_amdgcn_readfirstlane(sight.low), __builtin_amdgcn_readfirstlane(sight.sure_low)};
        }
        span = {0, 0, 0, 0};
        lo = round0 * kRound, hi = complete ? family.keys : min(family.keys, round1 * kRound);
        if (a.window > 0) seen_of_part<kSpanTile>(sight, &lo, &hi);
      } else {
        mine = seq.reach_of<SIGHT>(a, token);
        sight = sight_of(seq.reach_of<SIGHT>(a, token0), seq.reach_of<SIGHT>(a, token1));
      }
      if (of_family) {
      } else if constexpr (SIGHT) {
        span = span_of<kSpanTile>(sight, seq.base);
        lo = span.lo, hi = span.hi;
        if (!complete) {
          lo = span.lo + round0 * kRound;
          hi = min(hi, span.lo + round1 * kRound);
        }
      } else {
        lo = sight.first & ~(S::kKeys - 1), hi = sight.end;
        if (!complete) {
          lo = max(lo, (sight.first / kRound + round0) * kRound);
          hi = min(hi, (sight.first / kRound + round1) * kRound);
        }
      }
      auto key_at = [&](int place) __attribute__((always_inline)) {
        if constexpr (SIGHT) return span.key_at(place);
        else return place;
      };
      cursor.last = max(0, (sight.end - 1) >> view.page_shift);

      u32x4 qf[S::kSteps];
  #pragma unroll
      for (int i = 0; i < S::kSteps; ++i) {
        qf[i] = u32x4{0u, 0u, 0u, 0u};
        if (row < rows) qf[i] = *reinterpret_cast<const u32x4*>(q + (seq.start + token) * a.q_pitch + (int64_t)head * D + (quarter + 4 * i) * S::kElems);
      }
      floatx4 ot[S::kTiles];
  #pragma unroll
      for (int t = 0; t < S::kTiles; ++t) ot[t] = floatx4{0.f, 0.f, 0.f, 0.f};
      float top = -INFINITY, sum = 0.f;  // of scale * log2(e) * score; the sum is this quarter's share

      u32x4 kf[S::kGroups][S::kSteps], vf[S::kGroups][S::kValuePieces];
      auto load_keys = [&](int key) __attribute__((always_inline)) {
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          const T* p;
          if constexpr (!SMALL) p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(keys) + group_at<S::kRowBytes>(view, cursor, key + 16 * g)) + row * D;
          else p = keys + row_offset<D>(view, cursor, kv_head, key + 16 * g + row);
  #pragma unroll
          for (int i = 0; i < S::kSteps; ++i) kf[g][i] = *reinterpret_cast<const u32x4*>(p + (quarter + 4 * i) * S::kElems);
        }
      };
      auto load_values = [&](int key) __attribute__((always_inline)) {  // before the keys of the tile
        if constexpr (!SMALL) come_to<S::kRowBytes>(view, cursor, kv_head, key);
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          if constexpr (!SMALL) {
            const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(values) + group_at<S::kRowBytes>(view, cursor, key + 16 * g)) + lane * S::kElems;
  #pragma unroll
            for (int i = 0; i < S::kValuePieces; ++i) vf[g][i] = *reinterpret_cast<const u32x4*>(p + i * 64 * S::kElems);
          } else {
  #pragma unroll
            for (int i = 0; i < S::kValuePieces; ++i) {
              const int at = i * 1024 + lane * 16, r = at / S::kRowBytes;
              vf[g][i] = *reinterpret_cast<const u32x4*>(values + row_offset<D>(view, cursor, kv_head, key + 16 * g + r) + at % S::kRowBytes / (int)sizeof(T));
            }
          }
        }
      };

      constexpr int kStep = NW * S::kKeys;
      // One tile.  Whether another follows is known to the compiler: a load that may or may not have been sent would make it wait for all of them.
      auto work_on = [&](int place, auto more) __attribute__((always_inline)) {
        const int key = key_at(place);
        const bool masked = !all_see<SIGHT>(sight, key, S::kKeys) || place + S::kKeys > hi;
        uint32_t wild = 0;
        if (masked) {  // keys that no row sees may hold anything: their values count as zeros, and one that only some rows see must not reach the others
  #pragma unroll
          for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
            for (int i = 0; i < S::kValuePieces; ++i) {
              const int k = key + 16 * g + (i * 1024 + lane * 16) / S::kRowBytes;
              if (!some_see<SIGHT>(sight, k)) vf[g][i] = u32x4{0u, 0u, 0u, 0u};
              wild |= not_finite<T>(vf[g][i]);
            }
          wild = __any(wild != 0);
        }
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
          for (int i = 0; i < S::kValuePieces; ++i) {
            const int at = i * 1024 + lane * 16, r = 16 * g + at / S::kRowBytes;
            *reinterpret_cast<u32x4*>(tile + r * S::kRowBytes + value_piece<T, D>(r, at % S::kRowBytes / 16) * 16) = wild ? finite_part<T>(vf[g][i]) : vf[g][i];
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the tile is this wavefront's alone: its LDS accesses are in order)
        if constexpr (decltype(more)::value) load_values(key_at(place + kStep));

        floatx4 st[S::kGroups];
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          st[g] = floatx4{0.f, 0.f, 0.f, 0.f};
  #pragma unroll
          for (int i = 0; i < S::kSteps; ++i) st[g] = mma16<T>(kf[g][i], qf[i], st[g]);
        }
        if constexpr (decltype(more)::value) load_keys(key_at(place + kStep));
        if (masked) {
  #pragma unroll
          for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = key + 16 * g + 4 * quarter + e;
              if (!sees<SIGHT>(mine, k) || (!SIGHT && k >= hi)) st[g][e] = -INFINITY;  // (places end at hi with whole tiles, or with the last key)
            }
        }
        float m = st[0][0];
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
          for (int e = 0; e < 4; ++e) m = fmaxf(m, st[g][e]);
        const float moved = moved_reference(top, quarters_max(m) * a.scale_log2e);
        const float zero = moved == -INFINITY ? 0.f : moved;  // (a row that has seen no key yet)
        const float shrink = __builtin_amdgcn_exp2f(top - zero);
        top = moved;
        u32x4 pf{};
        float share = 0.f;
        float p[S::kGroups][4];
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
          for (int e = 0; e < 4; ++e) p[g][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[g][e], a.scale_log2e, -zero));
        if constexpr (sizeof(T) == 2) {
          // rounded to the type for the second product; the sum is that of the rounded ones, so what rounding does to all of them alike cancels
  #pragma unroll
          for (int w = 0; w < 4; ++w) {
            pf[w] = pack2<T>(p[w >> 1][2 * (w & 1)], p[w >> 1][2 * (w & 1) + 1]);
            share = add_pair<T>(pf[w], share);
          }
        } else {
  #pragma unroll
          for (int e = 0; e < 4; ++e) share += p[0][e];
        }
        sum = sum * shrink + share;
        if (__any(shrink != 1.f)) {
  #pragma unroll
          for (int t = 0; t < S::kTiles; ++t) ot[t] *= shrink;
        }
  #pragma unroll
        for (int t = 0; t < S::kTiles; ++t) {
          if constexpr (sizeof(T) == 2) {
            u32x4 v;
  #pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int r = 16 * g + 4 * quarter + (row >> 2);
              const u32x2 half = read_transposed(tile + r * S::kRowBytes + value_piece<T, D>(r, 2 * t + ((row >> 1) & 1)) * 16 + (row & 1) * 8);
              v[2 * g] = half[0], v[2 * g + 1] = half[1];
            }
            ot[t] = mma16<T>(v, pf, ot[t]);
          } else {
  #pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * quarter + e;
              const float v = *reinterpret_cast<const float*>(tile + r * S::kRowBytes + value_piece<T, D>(r, 4 * t + (row >> 2)) * 16 + (row & 3) * 4);
              ot[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[0][e], ot[t], 0, 0, 0);
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (wild) {  // a sum with an infinity or a NaN is one or the other
  #pragma unroll 1
          for (int k = key; k < (SIGHT ? key + S::kKeys : min(key + S::kKeys, hi)); ++k) {
            const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * quarter;
            const bool seen = sees<SIGHT>(mine, k);
  #pragma unroll
            for (int t = 0; t < S::kTiles; ++t)
  #pragma unroll
              for (int e = 0; e < 4; ++e) {
                float sum_e = ot[t][e];
                if (seen) add_wild(sum_e, v + 16 * t + e);
                ot[t][e] = sum_e;
              }
          }
        }
      };
      int place = lo + wave * S::kKeys;
      if (place < hi) {
        // (a wavefront's tiles lie kStep apart: behind the gap it begins anywhere in one of its steps, aligned as its tiles are)
        if constexpr (!SMALL && SIGHT) fetch_pages<S::kRowBytes>(view, cursor, kv_head, key_at(place), span.skip > 0 && place < span.seam ? span.seam + span.skip : 0);
        else if constexpr (!SMALL) fetch_pages<S::kRowBytes>(view, cursor, kv_head, place);
        load_values(key_at(place));
        load_keys(key_at(place));
        for (; place + kStep < hi; place += kStep) work_on(place, std::true_type{});
        work_on(place, std::false_type{});
      }

      // the wavefronts meet
      sum = quarters_sum(sum);
      __syncthreads();
      float* const stage = reinterpret_cast<float*>(smem);
  #pragma unroll
      for (int t = 0; t < S::kTiles; ++t)
        *reinterpret_cast<floatx4*>(stage + (wave * kFewRows + row) * S::kPitch + 16 * t + 4 * quarter) = ot[t];
      if (quarter == 0) met[wave][row][0] = top, met[wave][row][1] = sum;
      __syncthreads();
      {
        constexpr int kThreads = NW * 4, kWide = D / kThreads;  // of a row; columns of a thread
        const int r = tid / kThreads, d0 = tid % kThreads * kWide;
        if (r < rows) {
          float best = -INFINITY;
  #pragma unroll
          for (int w = 0; w < NW; ++w) best = fmaxf(best, met[w][r][0]);
          const float zero = best == -INFINITY ? 0.f : best;
          float total = 0.f, o[kWide] = {};
  #pragma unroll
          for (int w = 0; w < NW; ++w) {
            const float weight = __builtin_amdgcn_exp2f(met[w][r][0] - zero);
            total += met[w][r][1] * weight;
  #pragma unroll
            for (int c = 0; c < kWide; ++c) o[c] += stage[(w * kFewRows + r) * S::kPitch + d0 + c] * weight;
          }
          const int t = (row0 + r) / a.group, h = kv_head * a.group + row0 + r - t * a.group;
          if (complete && (!SIGHT || (seq.base == 0 && !of_family))) {
            const float inv = inverse_sum(total, seq.reach(a, t).end > 0);
            T* to = static_cast<T*>(a.out) + (seq.start + t) * a.out_pitch + (int64_t)h * D + d0;
            Vec<T, kWide> x;
  #pragma unroll
            for (int c = 0; c < kWide; ++c) x.v[c] = from_float<T>(o[c] * inv);
            store_vec<T, kWide>(to, x);
          } else {
            int64_t at = (2 * (int64_t)workgroup + (round0 == 0 ? 1 : 0)) * kFewRows + r;
            if (SIGHT && complete) {  // (of a family's: what it has in common, or of its own)
              const int64_t row_at = (seq.start + t) * (int64_t)a.heads + h;
              at = of_family ? a.family_at + row_at * a.family_splits : a.whole_at + row_at;
            }
            if (!of_family || shared.theirs[r]) {
              float* const ml = a.partial + (SIGHT ? a.rows : 2 * (int64_t)splits * kFewRows) * D + at * 2;
  #pragma unroll
              for (int c = 0; c < kWide; ++c) a.partial[at * D + d0 + c] = o[c];
              if (d0 == 0) ml[0] = best, ml[1] = total;
            }
          }
        }
      }
      if (row0 + kFewRows < rows_all || unit < stop) __syncthreads();
    }
  }
}

template <typename T, int D, int NW, bool SMALL, int SEES>
__global__ __launch_bounds__(NW * 64, 8 / NW) void few_rows_kernel(const PagedArgs a) {
  __shared__ FewRowsShared<T, D, NW> shared;
  Walk walk{};
  few_rows<T, D, NW, SMALL, SEES>(a, blockIdx.x, a.splits, walk, -1, shared);
}

// Which workgroups had a part of a pair: from first to last.
struct Sharers {
  int64_t first, last;
};
// `unit`: the first of the pair.
__device__ __forceinline__ Sharers sharers_of(int64_t unit, int rounds, int64_t units, int64_t workgroups) {
  return {quotient((unit + kStart + 1) * workgroups - 1, units), quotient((unit + rounds) * workgroups - 1, units)};
}

// Pairs that were several workgroups': their rows' partial results are joined, in 5 to 7 us, nearly all of them the launch and three trips to memory.  A workgroup per pair and row, or per pair where there are many of them: then a wavefront
// takes a row.
// us, a workgroup per row / per pair, 32 query and 8 key heads of 128: 1 sequence of 3000 keys 12.8 / 14.2, 8 (64 pairs) 24.9 / 25.4, 64 of 1500 (512) 75.4 / 73.8, 200 (1600)
// 241 / 228; 16 query heads of one key head, one sequence of 100000 keys beside 63 of 500, whose pair has most of the parts, 45.7 / 145.
constexpr int kManyPairs = 512;
template <typename T, int D, int SEES>
__global__ __launch_bounds__(256) void join_few_rows_kernel(const PagedArgs a, bool by_pair) {
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, b = blockIdx.x / view.kv_heads;
  const Sequence seq = sequence(a, b);  // (without families, whose parts are joined elsewhere)
  const int rows = seq.tokens * a.group;
  if (rows > a.few || (int)blockIdx.y >= rows) return;
  Walk walk{};
  const int64_t units = count_units<SEES>(a, walk), workgroups = sharers(a.splits, units);
  if (view.batch > kWave) walk_to_group<SEES>(a, walk, b / group_size(a));
  while (walk.base + kWave <= b) walk_on<SEES>(a, walk);
  const int lane = b - walk.base, rounds = __builtin_amdgcn_readlane(walk.rounds, lane);
  const Sharers shared = sharers_of(walk.before + lane_of(walk.upto, lane) - (int64_t)rounds * (view.kv_heads - kv_head), rounds, units, workgroups);
  const int64_t first = shared.first, last = shared.last;
  if (first == last) return;
  const int parts = (int)(last - first) + 1;
  const float* const ml = a.partial + (SEES != kWindow ? a.rows : 2 * (int64_t)a.splits * kFewRows) * D;
  auto sees = [&](int r) { return seq.reach(a, r / a.group).end > 0; };
  auto place = [&](int r) {
    const int t = r / a.group, h = kv_head * a.group + r - t * a.group;
    return static_cast<T*>(a.out) + (seq.start + t) * a.out_pitch + (int64_t)h * D;
  };
  if (by_pair) {
    for (int r = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r < rows; r += 4)
      join_parts_by_wavefront<T, D>(
          a.partial, ml, parts, sees(r), [&](int p) { return (2 * (first + p) + (p == 0 ? 1 : 0)) * kFewRows + r; }, place(r));
    return;
  }
  const int r = blockIdx.y;
  join_parts<T, D>(
      a.partial, ml, parts, sees(r), [&](int p) { return (2 * (first + p) + (p == 0 ? 1 : 0)) * kFewRows + r; }, place(r));
}

template <typename T, int D, int SEES>
void start_join_few_rows(const PagedArgs& a, hipStream_t stream) {
  if (a.splits == 0) return;
  const unsigned pairs = (unsigned)((int64_t)a.view.batch * a.view.kv_heads);
  const bool by_pair = pairs >= kManyPairs;
  hipLaunchKernelGGL((join_few_rows_kernel<T, D, SEES>), dim3(pairs, by_pair ? 1u : (unsigned)std::min<int64_t>(a.few, (int64_t)a.view.tokens * a.group)), dim3(256), 0,
                     stream, a, by_pair);
}
template <typename T, int SEES>
void start_few_rows(const PagedArgs& a, int64_t head_dim, hipStream_t stream) {
  const unsigned pairs = (unsigned)((int64_t)a.view.batch * a.view.kv_heads);
  const bool small = a.view.page_shift < 4;
  auto sized = [&](auto d) {
    constexpr int D = decltype(d)::value;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.splits > 0 ? (unsigned)a.splits : pairs), dim3(a.waves * 64), 0, stream, a); };
    if (small && a.waves == 4) launch(few_rows_kernel<T, D, 4, true, SEES>);
    else if (small) launch(few_rows_kernel<T, D, 8, true, SEES>);
    if constexpr (SEES != kFamilies) {  // (which are another launch's, but for small pages)
      if (!small && a.waves == 4) launch(few_rows_kernel<T, D, 4, false, SEES>);
      else if (!small) launch(few_rows_kernel<T, D, 8, false, SEES>);
      start_join_few_rows<T, D, SEES>(a, stream);
    }
  };
  if (head_dim == 64) sized(std::integral_constant<int, 64>{});
  else sized(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace ttmi
