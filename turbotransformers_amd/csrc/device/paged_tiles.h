// Attention over pages where sequences have many rows (new tokens times query heads of a key/value head): prompts and chunks of them.
//
// The matrix instructions bound it, and with them the exponentials and what LDS can feed.  A workgroup has 128 rows of one sequence and head, 32 a wavefront, and
// walks over tiles of 64 keys (fp32: 32) that all four share in LDS, fetched into registers one ahead and stored while the other stage is worked on.
// Scores are computed transposed, St[key, row] = K . Q^T (v_mfma_f32_32x32x16, fp32: 32x32x2), so a lane has one row, its statistics need one exchange of the two
// half-wavefronts, and the probabilities lie in the accumulators as Ot[d, row] += Vt . Pt wants them; Vt is what the transposing reads give of values that lie in LDS
// row by row as in the cache (fp32: plain reads of a column).  Packing a group's heads into one tile of rows reads the keys of a head once for all of them and keeps
// tiles full whatever the group.
//
// Measured, 32 query and 8 key heads of 128, bf16: a prompt of 8192 tokens 580 to 620 us (0.89 to 0.94 PFLOP/s; a large product here 1.26).  Of a SIMD's 1.19e6 cycles
// the matrix pipe is busy for 0.53e6 and vector instructions, the exponentials first, are at work for as many: the two hardly overlap.  Power comes second: on zeros the same launch takes 530 to 565 us.
// Heads of 64: 343 us (0.80), where an exponential takes a lane as long as its share of the products.  A workgroup by itself takes about 7 us to
// its first tile and 0.95 a tile of 64 keys, heads of 64, where four instructions' worth of products would be 0.2: a chain of reads, products, maximum, exponentials, products.
// The last blocks of a launch run on few CUs: 6 chunks of 400 to 600 tokens behind up to 9000 keys 220 us (0.85 PFLOP/s), 93 tiles for each of 512 places, 125 in the longest block.
// fp32 with heads of 128 has no registers left (256 and 96 bytes of scratch a lane): a prompt of 1000 tokens 153 us.
// What was built and taken out: 256 rows a workgroup with the products of 32 keys beside the exponentials of the 32 before, level to 3 % faster for heads of 128, 2 % slower for those of 64.
//
// THIRDS (fp32 with SIGHT): the fp32 instruction takes sixteen times as long as the bf16 one, so a number is a sum of three bf16, x = h + m + l to its last place, and a product six of theirs,
//     x y = h h' + (h m' + m h') + (m m' + h l' + l h'), up to 2^-23 of it left out (m is at most 2^-8, l 2^-16 of x);
// keys and values are taken apart on their way to LDS, queries once, probabilities as they come; sums are fp32 as ever.  Numbers from 2^127 on, whose h may be an infinity, have their scores
// computed one by one.  Where one that is not zero lies below 2^-100, whose l may be lost, the workgroup finds out while it takes them apart, and begins anew with the fp32 instruction (without the
// look for them: 8 prompts 33.5 us, one of 4000 104).  us, that instruction / this, 12 heads of 64: 8 prompts of 33 to 900 tokens, window 200 41.5 / 35.2, one of 4000, window 1000 171 / 109, 8 questions of
// 40 to 100 tokens behind 4000 common keys 94 / 70; 32 and 8 heads of 128: a prompt of 1000, window 300 125 / 74, 20 chunks of up to 300 behind up to 3000 keys 214 / 127.  Against 64 bits the error goes
// from 2.5e-7 to 1.8e-7.
//
// SIGHT: rows that see the first keys of their sequence besides a window (the keys that a block sees lie behind each other in whole tiles, Span), sequences whose first keys are their family's,
// and families: the rows of all sequences of one over the keys that they have in common, each of which sees what its own position lets it see.
#pragma once

#include "paged_attention.h"

namespace ttmi {
namespace {

constexpr int kTileRows = 128;  // of a workgroup
template <typename T>
constexpr int kSpanTiles = sizeof(T) == 2 ? 64 : 32;
// Parts that a row's own keys lie in (1 where it sees none of them).
__device__ __forceinline__ int own_parts(const Reach& r, const Span& span, int base, int chunk) {
  return r.end > base ? (span.place_of(r.end - 1) - span.lo) / chunk + 1 : 1;
}

template <typename T, int D>
struct Tiles {
  static constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // (as in kSpanTiles)
  static constexpr int kSubs = kKeys / 32;
  static constexpr int kElems = 16 / (int)sizeof(T);
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kBytes = kKeys * kRowBytes;      // of a tile of keys, or of values
  static constexpr int kPieces = kBytes / 4096;         // 16-byte pieces of a tile per thread
  static constexpr int kSteps = kRowBytes / 32;         // pieces of a row per lane, for the first product
  static constexpr int kOut = D / 32;
  // Tiles on their way in registers.  us, 6 chunks of 400 to 600 tokens behind 1500 to 9000 keys, 32 query and 8 key heads of 64, one / two: fp32 936 / 838, bf16 151 / 154
  // (head_dim 128 has no registers for two).
  static constexpr int kDepth = sizeof(T) == 4 && D == 64 ? 2 : 1;
};

// Places of a row's 16-byte pieces in LDS.  Keys: sixteen rows read the same piece at a time.  Values: 64 bytes of four rows at a time (fp32: 128 bytes of two rows that lie
// four apart).  The exclusive or takes them to different banks.
template <typename T, int D>
__device__ __forceinline__ int key_piece(int row, int piece) {
  if constexpr (sizeof(T) == 2 && D == 64) return piece ^ ((row >> 1) & 7);
  else return piece ^ (row & 15);
}
template <typename T, int D>
__device__ __forceinline__ int tile_value_piece(int row, int piece) {
  if constexpr (sizeof(T) == 4) return piece ^ (((row >> 2) & 1) << 3);
  else if constexpr (D == 128) return piece ^ ((row & 3) << 2);
  else return piece ^ (((row >> 1) & 1) << 2);
}

// A row's sums, divided and stored.
template <typename T, int D>
__device__ __forceinline__ void store_out(const PagedArgs& a, int64_t token, int head, bool sees, int lhalf, const floatx16 (&ot)[D / 32], float sum) {
  const float inv = inverse_sum(sum, sees);
  T* to = static_cast<T*>(a.out) + token * a.out_pitch + (int64_t)head * D + 4 * lhalf;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      Vec<T, 4> x;
#pragma unroll
      for (int c = 0; c < 4; ++c) x.v[c] = from_float<T>(ot[t][4 * g + c] * inv);
      store_vec<T, 4>(to + 32 * t + 8 * g, x);
    }
}
// The same where the row's keys lie in several parts: kept for the kernel that joins those, in row `at` of `rows` partial results.
template <int D>
__device__ __forceinline__ void store_part(const PagedArgs& a, int64_t at, int64_t rows, int lhalf, const floatx16 (&ot)[D / 32], float top, float sum) {
  float* to = a.partial + at * D + 4 * lhalf;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<floatx4*>(to + 32 * t + 8 * g) = floatx4{ot[t][4 * g], ot[t][4 * g + 1], ot[t][4 * g + 2], ot[t][4 * g + 3]};
  if (lhalf == 0) {
    float* ml = a.partial + rows * D + at * 2;
    ml[0] = top, ml[1] = sum;
  }
}

// The `want`-th block of rows of all sequences -> its sequence and number in it (false: there are fewer).  Every lane looks at a sequence of 64.
// Where there are more workgroups than the chip takes at a time, those with the most keys come first: sequences by their keys (64 of them at a time), and in a sequence the
// last rows, which have the most keys before them.
__device__ __forceinline__ bool find_block(const PagedArgs& a, int want, int* b, int* block) {
  const int lane = (int)(threadIdx.x % kWave);
  for (int base = 0; base < a.view.batch; base += kWave) {
    int blocks = 0, reach = 0;
    if (base + lane < a.view.batch) {
      const Sequence seq = sequence(a, base + lane);
      const int rows = seq.tokens * a.group;
      if (rows > kFewRows || a.every) blocks = (rows + kTileRows - 1) / kTileRows;
      reach = a.window > 0 ? min(seq.length, a.window + seq.tokens) : seq.length;
    }
    int before = 0, all = 0;
    if (!a.ordered) {
      int upto = blocks;
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) {
        const int below = __shfl_up(upto, d, kWave);
        if (lane >= d) upto += below;
      }
      before = upto - blocks, all = __builtin_amdgcn_readlane(upto, kWave - 1);
    } else {
      for (uint64_t others = __ballot(blocks > 0); others != 0; others &= others - 1) {
        const int j = __ffsll((unsigned long long)others) - 1;
        const int their_blocks = __builtin_amdgcn_readlane(blocks, j), their_reach = __builtin_amdgcn_readlane(reach, j);
        all += their_blocks;
        if (their_reach > reach || (their_reach == reach && j < lane)) before += their_blocks;
      }
    }
    if (want < all) {
      const int found = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(want >= before && want < before + blocks)) - 1);
      *b = base + found;
      *block = __builtin_amdgcn_readlane(before + blocks, found) - 1 - want;
      return true;
    }
    want -= all;
  }
  return false;
}

// Four floats as sums of three bf16 each, whose products the bf16 instructions add up 16 keys at a time.
struct Thirds {
  u32x2 part[3];
};
__device__ __forceinline__ Thirds thirds(const u32x4& raw) {
  const floatx4 x = __builtin_bit_cast(floatx4, raw);
  Thirds t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t both = pack2<bf16>(a, b);
      t.part[p][i] = both;
      a -= __builtin_bit_cast(float, both << 16), b -= __builtin_bit_cast(float, both & 0xffff0000u);
    }
  }
  return t;
}
// Numbers that this cannot take apart: their bf16 may be an infinity, times which the other parts would be NaN.
constexpr float kTooLarge = 0x1p127f;
__device__ __forceinline__ bool too_large(const u32x4& raw) {
  const floatx4 x = __builtin_bit_cast(floatx4, raw);
  return fmaxf(fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])), fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3]))) >= kTooLarge;
}

// And those whose last part lies below bf16's normal numbers (2^-126 for a last place of 2^-123), zero apart.  least: the least of what was looked at so far, as a magnitude's bits
// twice and less one.
constexpr uint32_t kTooSmall = 2 * 0x0d800000u - 1;  // 2^-100
__device__ __forceinline__ uint32_t least_of(uint32_t least, const u32x4& raw) {
#pragma unroll
  for (int i = 0; i < 4; ++i) least = min(least, (raw[i] << 1) - 1u);
  return least;
}

template <typename T, int D, bool THIRDS>
struct TilesShared {
  static constexpr int kBytes = THIRDS ? Tiles<T, D>::kBytes * 3 / 2 : Tiles<T, D>::kBytes;  // of a tile of keys, or of values
  __align__(16) char tiles[4 * kBytes];
  int wild;  // whether values that only some rows see hold infinities or NaNs
  int large;  // THIRDS: whether a key was too large
  int small;  // THIRDS: whether a number was too small
  int sights[4][6];  // of a family's rows, wavefront by wavefront
};

// What the rows of a family that a wavefront's lanes have see (`live`: this lane has one), and what all rows of the workgroup do.  Mostly everything.
template <typename Shared>
__device__ __forceinline__ void family_sights(const Family& f, const Reach& mine, bool live, int wave, Shared& shared, Sight* of_wave, Sight* of_all) {
  Sight s = {0, f.keys, 0, f.keys, 0, 0};
  if (!__all(!live || (mine.begin == 0 && mine.end == f.keys && mine.low == 0))) {
    s.first = live ? mine.begin : INT32_MAX, s.end = live ? mine.end : 0, s.sure_first = live ? mine.begin : 0, s.sure_end = live ? mine.end : INT32_MAX;
    s.low = live ? mine.low : 0, s.sure_low = live ? mine.low : INT32_MAX;
#pragma unroll 1
    for (int d = 1; d < kWave; d *= 2) {
      s.first = min(s.first, __shfl_xor(s.first, d, kWave)), s.end = max(s.end, __shfl_xor(s.end, d, kWave));
      s.sure_first = max(s.sure_first, __shfl_xor(s.sure_first, d, kWave)), s.sure_end = min(s.sure_end, __shfl_xor(s.sure_end, d, kWave));
      s.low = max(s.low, __shfl_xor(s.low, d, kWave)), s.sure_low = min(s.sure_low, __shfl_xor(s.sure_low, d, kWave));
    }
    s = {__builtin_amdgcn_readfirstlane(s.first), __builtin_amdgcn_readfirstlane(s.end), __builtin_amdgcn_readfirstlane(s.sure_first),
         __builtin_amdgcn_readfirstlane(s.sure_end), __builtin_amdgcn_readfirstlane(s.low), __builtin_amdgcn_readfirstlane(s.sure_low)};
  } else if (!__any(live)) s = {INT32_MAX, 0, 0, INT32_MAX, 0, INT32_MAX};
  *of_wave = s;
  const int lane = (int)(threadIdx.x % kWave);
  if (lane == 0) {
    int* const to = shared.sights[wave];
    to[0] = s.first, to[1] = s.end, to[2] = s.sure_first, to[3] = s.sure_end, to[4] = s.low, to[5] = s.sure_low;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int* const from = shared.sights[w];
    s.first = min(s.first, from[0]), s.end = max(s.end, from[1]), s.sure_first = max(s.sure_first, from[2]), s.sure_end = min(s.sure_end, from[3]);
    s.low = max(s.low, from[4]), s.sure_low = min(s.sure_low, from[5]);
  }
  *of_all = {__builtin_amdgcn_readfirstlane(s.first), __builtin_amdgcn_readfirstlane(s.end), __builtin_amdgcn_readfirstlane(s.sure_first),
             __builtin_amdgcn_readfirstlane(s.sure_end), __builtin_amdgcn_readfirstlane(s.low), __builtin_amdgcn_readfirstlane(s.sure_low)};
}

// Part `z` of a block of rows of sequence b; SIGHT: of the sequence's own keys, or (family.keys > 0) of the family's that it leads, in parts of family_chunk keys.
// SMALL: pages of fewer than 16 slots
// THIRDS: fp32 by the bf16 instructions.  -> false where a number was too small for that: nothing is stored then, and the part is one for the fp32 instruction
template <typename T, int D, bool SMALL, bool SIGHT, bool FAMILIES, bool THIRDS>
__device__ __forceinline__ bool tiles(const PagedArgs& a, int b, int block, const Sequence& seq, const LaneSequences& lanes, const Family& family, int family_chunk,
                                      int kv_head, int z, int tid, TilesShared<T, D, THIRDS>& shared) {
  using S = Tiles<T, D>;
  constexpr int kTileBytes = TilesShared<T, D, THIRDS>::kBytes, kPlane = kTileBytes / 3;  // (THIRDS: of a third of the tile)
  char* const smem = shared.tiles;
  int& wild = shared.wild;
  const PagedView& view = a.view;
  const bool families = FAMILIES && family.keys > 0;
  const int row0 = block * kTileRows, rows = min(kTileRows, seq.tokens * a.group - row0);
  if (z == 0 && kv_head == 0 && block == 0 && tid == 0 && !families && seq.first + seq.tokens > seq.length) page_error(view);

  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lrow = lane & 31, lhalf = lane >> 5;
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  const int wave_rows = max(0, min(32, rows - wave * 32));
  const int wrow = row0 + wave * 32;
  bool live = lrow < wave_rows;
  const int token = (wrow + (live ? lrow : 0)) / a.group, head = kv_head * a.group + (live ? wrow + lrow - token * a.group : 0);
  // what the rows of the workgroup see, and those of this wavefront
  Reach mine;
  Sight sight, wave_sight;
  if (families) {
    bool member;
    mine = family_reach(a, lanes, family, seq.start, seq.start + (wave_rows > 0 ? token : 0), &member);
    live = live && member;  // (others' rows are not this family's, whatever it says)
    family_sights(family, mine, live, wave, shared, &wave_sight, &sight);
  } else {
    mine = seq.reach_of<SIGHT>(a, token);
    sight = sight_of(seq.reach_of<SIGHT>(a, row0 / a.group), seq.reach_of<SIGHT>(a, (row0 + rows - 1) / a.group));
    wave_sight = sight_of(seq.reach_of<SIGHT>(a, wrow / a.group), seq.reach_of<SIGHT>(a, (wrow + max(wave_rows, 1) - 1) / a.group));
    if (wave_rows <= 0) wave_sight.end = wave_sight.low = 0;
  }
  // its part of them; SIGHT: places
  int chunk, part0, part, lo, hi;
  Span span;
  if constexpr (!SIGHT) {
    chunk = seq.chunk(a);
    part0 = sight.first / chunk, part = part0 + z;
    lo = (int)max(part * (int64_t)chunk, (int64_t)(sight.first & ~(S::kKeys - 1))), hi = (int)min((part + 1) * (int64_t)chunk, (int64_t)sight.end);
    if (lo >= hi && part != part0) return true;
  } else {
    part0 = 0, part = z;
    if (families) {  // all rows of a family have the same parts, and write them
      chunk = family_chunk;
      span = {0, 0, 0, 0};
      if (z * (int64_t)chunk >= seq.length) return true;
      lo = z * chunk, hi = (int)min((z + 1) * (int64_t)chunk, (int64_t)seq.length);
      if (a.window > 0) seen_of_part<S::kKeys>(sight, &lo, &hi);
    } else {
      chunk = seq.span_chunk(a);
      span = span_of<kSpanTiles<T>>(sight, seq.base);
      lo = (int)min(span.lo + part * (int64_t)chunk, (int64_t)span.hi), hi = (int)min(span.lo + (part + 1) * (int64_t)chunk, (int64_t)span.hi);
      if (lo >= hi && part != 0) return true;
    }
  }
  auto key_at = [&](int place) __attribute__((always_inline)) {
    if constexpr (SIGHT) return span.key_at(place);
    else return place;
  };

  const T* const query = static_cast<const T*>(a.q) + (seq.start + token) * a.q_pitch + (int64_t)head * D;
  u32x4 qf[THIRDS ? 1 : S::kSteps], qt[THIRDS ? 3 : 1][D / 16];
  bool large_query = false;
  uint32_t least = UINT32_MAX;  // THIRDS: of this lane's share of what the workgroup reads and some row sees
  if constexpr (!THIRDS) {
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
      qf[i] = u32x4{0u, 0u, 0u, 0u};
      if (live) qf[i] = *reinterpret_cast<const u32x4*>(query + (2 * i + lhalf) * S::kElems);
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (live) x = *reinterpret_cast<const u32x4*>(query + 16 * i + 8 * lhalf + 4 * j);
        large_query = large_query || too_large(x), least = least_of(least, x);
        const Thirds t = thirds(x);
#pragma unroll
        for (int p = 0; p < 3; ++p) qt[p][i][2 * j] = t.part[p][0], qt[p][i][2 * j + 1] = t.part[p][1];
      }
    large_query = __shfl_xor((int)large_query, 32, kWave) != 0 || large_query;  // (the row's other half)
  }
  floatx16 ot[S::kOut];
#pragma unroll
  for (int t = 0; t < S::kOut; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) ot[t][e] = 0.f;
  float top = -INFINITY, sum = 0.f;

  typename std::conditional<SIGHT, GapCursor, PageCursor>::type cursor;
  cursor.table = view.table + (int64_t)b * view.table_pitch;
  cursor.last = max(0, (sight.end - 1) >> view.page_shift);
  cursor.first = 0, cursor.ahead = 0, cursor.at = 0;
  u32x4 kr[S::kDepth][S::kPieces], vr[S::kDepth][S::kPieces];
  // 16-byte pieces of a tile: thread by thread, 4 KB after 4 KB.  A wavefront's 1 KB lies in one group of 16 rows.
  auto load_piece = [&](int i, int key, int set) __attribute__((always_inline)) {
    if constexpr (!SMALL) {
      const int group = (i * 4096 + wave * 1024) / (16 * S::kRowBytes) * 16;
      const int64_t from = group_at<S::kRowBytes>(view, cursor, key + group);
      const uint32_t in_group = (uint32_t)(i * 4096 + tid * 16) % (16 * S::kRowBytes);
      kr[set][i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(keys) + from + in_group);
      vr[set][i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(values) + from + in_group);
    } else {
      const int at = i * 4096 + tid * 16;
      const int64_t from = row_offset<D>(view, cursor, kv_head, key + at / S::kRowBytes) + at % S::kRowBytes / (int)sizeof(T);
      kr[set][i] = *reinterpret_cast<const u32x4*>(keys + from);
      vr[set][i] = *reinterpret_cast<const u32x4*>(values + from);
    }
  };
  auto key_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * kTileBytes; };
  auto value_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * kTileBytes + kTileBytes; };
  auto store_piece = [&](int i, int s, int set) __attribute__((always_inline)) {
    const int at = i * 4096 + tid * 16, r = at / S::kRowBytes, c = at % S::kRowBytes / 16;
    if constexpr (THIRDS) {
      if (__builtin_expect(too_large(kr[set][i]), 0)) shared.large = 1;
      least = least_of(least_of(least, kr[set][i]), vr[set][i]);
      const Thirds k = thirds(kr[set][i]), v = thirds(vr[set][i]);
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        *reinterpret_cast<u32x2*>(key_stage(s) + p * kPlane + r * 2 * D + key_piece<bf16, D>(r, c / 2) * 16 + c % 2 * 8) = k.part[p];
        *reinterpret_cast<u32x2*>(value_stage(s) + p * kPlane + r * 2 * D + tile_value_piece<bf16, D>(r, c / 2) * 16 + c % 2 * 8) = v.part[p];
      }
      return;
    }
    *reinterpret_cast<u32x4*>(key_stage(s) + r * S::kRowBytes + key_piece<T, D>(r, c) * 16) = kr[set][i];
    *reinterpret_cast<u32x4*>(value_stage(s) + r * S::kRowBytes + tile_value_piece<T, D>(r, c) * 16) = vr[set][i];
  };
  // Keys that no row sees may hold anything: their values count as zeros.  Where only some rows see a key, infinities and NaNs of its values must not
  // reach the others: they are left out here, noted, and added where they are seen.
  auto partly_seen = [&](int key) __attribute__((always_inline)) { return !all_see<SIGHT>(sight, key, S::kKeys); };
  auto clean_values = [&](int key, int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int k = key + (i * 4096 + tid * 16) / S::kRowBytes;
      const bool seen = some_see<SIGHT>(sight, k);
      if (!seen) vr[set][i] = u32x4{0u, 0u, 0u, 0u};
      if (THIRDS && !seen) kr[set][i] = u32x4{0u, 0u, 0u, 0u};  // (or one that is too large would have its tile's scores looked at one by one)
      if (not_finite<T>(vr[set][i])) wild = 1;
      vr[set][i] = finite_part<T>(vr[set][i]);
    }
  };
  if (lo < hi) {
    // (Loads past the last tile fetch that once more, out of L2: a load that may or may not have been sent would make the compiler wait for all of them.)
    const int last = lo + (hi - 1 - lo) / S::kKeys * S::kKeys;
    if constexpr (!SMALL && SIGHT) fetch_pages<S::kRowBytes>(view, cursor, kv_head, key_at(lo), span.skip > 0 && lo < span.seam ? span.seam + span.skip : 0);
    else if constexpr (!SMALL) fetch_pages<S::kRowBytes>(view, cursor, kv_head, lo);
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) load_piece(i, key_at(lo), 0);
    if (tid == 0) wild = 0, shared.large = shared.small = 0;
    __syncthreads();
    if (partly_seen(key_at(lo))) clean_values(key_at(lo), 0);
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) store_piece(i, 0, 0);
#pragma unroll
    for (int n = 1; n <= S::kDepth; ++n) {
      const int next = key_at(min(lo + n * S::kKeys, last));
      if constexpr (SIGHT && !SMALL) come_to<S::kRowBytes>(view, cursor, kv_head, next);
#pragma unroll
      for (int i = 0; i < S::kPieces; ++i) load_piece(i, next, n % S::kDepth);  // (in the same 64 pages, or SIGHT behind a gap)
    }
    __syncthreads();
    // One tile; its stage is known to the compiler, so that places in LDS are fixed numbers behind one of the lane's.
    auto work_on = [&](int place, auto stage) __attribute__((always_inline)) {
      constexpr int s = decltype(stage)::value;
      const int key = key_at(place);
      // The other stage is free: what was fetched for it while the last tile was worked on goes there, and the tile behind it is sent for.
      constexpr int set = (s + 1) % S::kDepth;
      const int after = key_at(min(place + (1 + S::kDepth) * S::kKeys, last));
      if constexpr (!SMALL) come_to<S::kRowBytes>(view, cursor, kv_head, after);
      if (__builtin_expect(partly_seen(key_at(place + S::kKeys)), 0)) clean_values(key_at(place + S::kKeys), set);
      if ((key >= wave_sight.end || key + S::kKeys <= wave_sight.first) && (!SIGHT || key >= wave_sight.low)) {  // nothing to do for this wavefront's rows
#pragma unroll
        for (int i = 0; i < S::kPieces; ++i) store_piece(i, s ^ 1, set);
#pragma unroll
        for (int i = 0; i < S::kPieces; ++i) load_piece(i, after, set);
        __syncthreads();
        return;
      }
      const char* const kt = key_stage(s);
      const char* const vt = value_stage(s);
      floatx16 st[S::kSubs];
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[u][e] = 0.f;
      // Reads run kAhead instructions before their use.  The fences keep that order: left to itself the compiler waits for each read in front of its use.
      constexpr int kAhead = 4;
      u32x4 f[kAhead];
      if constexpr (!THIRDS) {
        auto read_keys = [&](int n) __attribute__((always_inline)) {  // the operand of the n-th matrix instruction of St
          const int r = 32 * (n % S::kSubs) + lrow;
          return *reinterpret_cast<const u32x4*>(kt + r * S::kRowBytes + key_piece<T, D>(r, 2 * (n / S::kSubs) + lhalf) * 16);
        };
        constexpr int kScores = S::kSubs * S::kSteps;
#pragma unroll
        for (int n = 0; n < kAhead; ++n) f[n] = read_keys(n);
#pragma unroll
        for (int n = 0; n < kScores; ++n) {
          st[n % S::kSubs] = mma32<T>(f[n % kAhead], qf[n / S::kSubs], st[n % S::kSubs]);
          if (n + kAhead < kScores) f[n % kAhead] = read_keys(n + kAhead);
          if (n < S::kPieces) store_piece(n, s ^ 1, set);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        // products of the parts, the small ones in a sum of their own (those of the smallest with each other and with the middle ones are less than what fp32 rounds)
        floatx16 small = st[0];
        u32x4 k[2][3];
        auto read_keys = [&](int i, int p) __attribute__((always_inline)) {
          return *reinterpret_cast<const u32x4*>(kt + p * kPlane + lrow * 2 * D + key_piece<bf16, D>(lrow, 2 * i + lhalf) * 16);
        };
#pragma unroll
        for (int p = 0; p < 3; ++p) k[0][p] = read_keys(0, p);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          if (i + 1 < D / 16) {
#pragma unroll
            for (int p = 0; p < 3; ++p) k[(i + 1) % 2][p] = read_keys(i + 1, p);
          }
          const u32x4(&x)[3] = k[i % 2];
          small = mma32<bf16>(x[2], qt[0][i], small);
          st[0] = mma32<bf16>(x[1], qt[0][i], st[0]);
          small = mma32<bf16>(x[0], qt[2][i], small);
          st[0] = mma32<bf16>(x[0], qt[1][i], st[0]);
          small = mma32<bf16>(x[1], qt[1][i], small);
          st[0] = mma32<bf16>(x[0], qt[0][i], st[0]);
          if (i < S::kPieces) store_piece(i, s ^ 1, set);
          __builtin_amdgcn_sched_barrier(0);
        }
        st[0] += small;
        // (scores of too large numbers, and no others, element by element)
        if (__builtin_expect(__any(large_query) || shared.large, 0)) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const T* const row = keys + row_offset<D>(view, cursor, kv_head, key + 8 * (e / 4) + 4 * lhalf + e % 4);
            float score = 0.f;
            bool large = large_query;
            if (live) {
#pragma unroll 1
              for (int d = 0; d < D; ++d) score = __builtin_fmaf(row[d], query[d], score), large = large || __builtin_fabsf(row[d]) >= kTooLarge;
            }
            st[0][e] = large ? score : st[0][e];
            __builtin_amdgcn_sched_barrier(0);  // (few registers: this path is cold)
          }
        }
      }
#pragma unroll
      for (int i = 0; i < S::kPieces; ++i) load_piece(i, after, set);
      if (__builtin_expect(!all_see<SIGHT>(wave_sight, key, S::kKeys), 0)) {
        // (a tile below `low` may have a hole behind what is seen of the first keys: then what is seen in it ends with the rest, and the hole is taken out)
        const bool holed = SIGHT && key < wave_sight.low;
        const int begin = holed ? min(mine.begin, key) : mine.begin, from = begin - key - 4 * lhalf;
        const uint32_t span = (uint32_t)(mine.end - begin);
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((uint32_t)(32 * u + 8 * (e / 4) + e % 4 - from) >= span) st[u][e] = -INFINITY;
        if (holed) {
          const int hole = mine.low - key - 4 * lhalf;
          const uint32_t keys = (uint32_t)max(0, mine.begin - mine.low);
#pragma unroll
          for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if ((uint32_t)(32 * u + 8 * (e / 4) + e % 4 - hole) < keys) st[u][e] = -INFINITY;
        }
      }
      float m;
      {
        float part[4];  // (chains of a quarter of the length)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          part[j] = st[0][j];
#pragma unroll
          for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
            for (int e = j; e < 16; e += 4) part[j] = fmaxf(part[j], st[u][e]);
        }
        const LanePair sw = swap_halves(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
        m = fmaxf(sw.a, sw.b);
      }
      const float moved = moved_reference(top, m * a.scale_log2e);
      const float zero = moved == -INFINITY ? 0.f : moved;  // (a row that has seen no key yet)
      const float shrink = __builtin_amdgcn_exp2f(top - zero);
      top = moved;
      if (__builtin_expect(__any(shrink != 1.f), 0)) {
        sum *= shrink;
#pragma unroll
        for (int t = 0; t < S::kOut; ++t) ot[t] *= shrink;
      }
      if constexpr (sizeof(T) == 2) {
        auto read_values = [&](int n) __attribute__((always_inline)) {  // the operand of the n-th matrix instruction of Ot: kOut of them for each 16 keys
          const int r0 = 16 * (n / S::kOut) + 4 * lhalf + ((lane >> 2) & 3), t = n % S::kOut;
          u32x4 v;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int r = r0 + 8 * g;
            const u32x2 half = read_transposed(vt + r * S::kRowBytes + tile_value_piece<T, D>(r, 4 * t + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8);
            v[2 * g] = half[0], v[2 * g + 1] = half[1];
          }
          return v;
        };
        // Probabilities, rounded to the type for the second product; their sum is that of the rounded ones, so what rounding does to all of them alike cancels.  Eight
        // of a row's at a time are what a lane gives the instructions of 16 keys.
        u32x4 pf[2 * S::kSubs];
        auto probabilities = [&](int pair) __attribute__((always_inline)) {
          float p[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[pair / 8][2 * (pair % 8) + j], a.scale_log2e, -zero));
          pf[pair / 4][pair % 4] = pack2<T>(p[0], p[1]);
          sum = add_pair<T>(pf[pair / 4][pair % 4], sum);
        };
        constexpr int kProducts = 2 * S::kSubs * S::kOut, kPairs = 8 * S::kSubs, kFirst = 4;
#pragma unroll
        for (int n = 0; n < kAhead; ++n) f[n] = read_values(n);
#pragma unroll
        for (int n = 0; n < kFirst; ++n) probabilities(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kProducts; ++n) {
          ot[n % S::kOut] = mma32<T>(f[n % kAhead], pf[n / S::kOut], ot[n % S::kOut]);
          if (n + kAhead < kProducts) f[n % kAhead] = read_values(n + kAhead);
          // the next 16 keys' probabilities beside this 16 keys' instructions
          if (n / S::kOut + 1 < 2 * S::kSubs) {
            constexpr int kEach = 4 / S::kOut;
#pragma unroll
            for (int j = 0; j < kEach; ++j) probabilities(kFirst + n * kEach + j);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else if constexpr (THIRDS) {
        u32x4 pt[3][2];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          floatx4 p;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][4 * g + j], a.scale_log2e, -zero));
            sum += p[j];
          }
          const Thirds t = thirds(__builtin_bit_cast(u32x4, p));
#pragma unroll
          for (int n = 0; n < 3; ++n) pt[n][g / 2][g % 2 * 2] = t.part[n][0], pt[n][g / 2][g % 2 * 2 + 1] = t.part[n][1];
        }
        auto read_values = [&](int n, int p) __attribute__((always_inline)) {  // kOut operands for each 16 keys
          const int r0 = 16 * (n / S::kOut) + 4 * lhalf + ((lane >> 2) & 3), t = n % S::kOut;
          u32x4 v;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int r = r0 + 8 * g;
            const u32x2 half =
                read_transposed(vt + p * kPlane + r * 2 * D + tile_value_piece<bf16, D>(r, 4 * t + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8);
            v[2 * g] = half[0], v[2 * g + 1] = half[1];
          }
          return v;
        };
        u32x4 v[2][3];
#pragma unroll
        for (int p = 0; p < 3; ++p) v[0][p] = read_values(0, p);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 2 * S::kOut; ++n) {
          if (n + 1 < 2 * S::kOut) {
#pragma unroll
            for (int p = 0; p < 3; ++p) v[(n + 1) % 2][p] = read_values(n + 1, p);
          }
          const u32x4(&x)[3] = v[n % 2];
          floatx16& to = ot[n % S::kOut];
          const int g = n / S::kOut;
          to = mma32<bf16>(x[2], pt[0][g], to);
          to = mma32<bf16>(x[0], pt[2][g], to);
          to = mma32<bf16>(x[1], pt[1][g], to);
          to = mma32<bf16>(x[1], pt[0][g], to);
          to = mma32<bf16>(x[0], pt[1][g], to);
          to = mma32<bf16>(x[0], pt[0][g], to);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        static_assert(sizeof(T) == 2 || S::kSubs == 1, "32 keys");
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          st[0][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][e], a.scale_log2e, -zero));
          sum += st[0][e];
        }
        auto read_value = [&](int n) __attribute__((always_inline)) {  // the operand of the n-th matrix instruction of Ot: kOut of them for each pair of keys
          const int e = n / S::kOut, r = 8 * (e / 4) + 4 * lhalf + e % 4;
          return *reinterpret_cast<const float*>(vt + r * S::kRowBytes + tile_value_piece<T, D>(r, 8 * (n % S::kOut) + (lrow >> 2)) * 16 + (lrow & 3) * 4);
        };
        constexpr int kProducts = 16 * S::kOut;
        float v[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) v[n] = read_value(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kProducts; ++n) {
          ot[n % S::kOut] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[n % kAhead], st[0][n / S::kOut], ot[n % S::kOut], 0, 0, 0);
          if (n + kAhead < kProducts) v[n % kAhead] = read_value(n + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (__builtin_expect(partly_seen(key), 0) && wild) {  // a sum with an infinity or a NaN is one or the other
#pragma unroll 1
        for (int k = key; k < (SIGHT ? key + S::kKeys : min(key + S::kKeys, hi)); ++k) {
          const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * lhalf;
          const bool seen = sees<SIGHT>(mine, k);
#pragma unroll
          for (int t = 0; t < S::kOut; ++t) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float sum_e = ot[t][e];
              if (seen) add_wild(sum_e, v + 32 * t + 8 * (e / 4) + e % 4);
              ot[t][e] = sum_e;
            }
            __builtin_amdgcn_sched_barrier(0);  // (few registers: this path is cold)
          }
        }
      }
      __syncthreads();
    };
    // (the last one stores that which was fetched once more, which nothing is asked about)
    auto count = [&](int place, auto stage) __attribute__((always_inline)) {
      const uint32_t before = least;
      work_on(place, stage);
      if constexpr (THIRDS) least = place + S::kKeys < hi ? least : before;
    };
    for (int place = lo; place < hi; place += 2 * S::kKeys) {
      count(place, std::integral_constant<int, 0>{});
      if (place + S::kKeys < hi) count(place + S::kKeys, std::integral_constant<int, 1>{});
    }
    if constexpr (THIRDS) {
      if (__builtin_expect(least < kTooSmall, 0)) shared.small = 1;
      __syncthreads();
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(shared.small), 0)) return false;
    }
  }

  {
    const LanePair both = swap_halves(sum);
    sum = both.a + both.b;
  }
  if (!live) return true;
  const int64_t at_token = seq.start + token;
  if constexpr (!SIGHT) {
    const bool sees_some = mine.end > 0;
    const int first_part = sees_some ? mine.begin / chunk : part0, last_part = sees_some ? (mine.end - 1) / chunk : part0;
    if (first_part == last_part) {
      if (part == first_part) store_out<T, D>(a, at_token, head, sees_some, lhalf, ot, sum);
    } else store_part<D>(a, (at_token * a.heads + head) * a.splits + part % a.splits, (int64_t)view.tokens * a.heads * a.splits, lhalf, ot, top, sum);
  } else if (families) store_part<D>(a, a.family_at + (at_token * a.heads + head) * a.family_splits + part, a.rows, lhalf, ot, top, sum);
  else {
    const int last_part = own_parts(mine, span, seq.base, chunk) - 1;
    if (last_part == 0 && seq.base == 0) {
      if (part == 0) store_out<T, D>(a, at_token, head, mine.end > 0, lhalf, ot, sum);
    } else if (part <= last_part) store_part<D>(a, a.own_at + (at_token * a.heads + head) * a.splits + part, a.rows, lhalf, ot, top, sum);
  }
  return true;
}

template <typename T, int D, bool SMALL>
__global__ __launch_bounds__(256, 2) void tiles_kernel(const PagedArgs a) {
  __shared__ TilesShared<T, D, false> shared;
  const int kv_head = blockIdx.x % a.view.kv_heads;
  int b, block;
  if (!find_block(a, blockIdx.x / a.view.kv_heads, &b, &block)) return;
  tiles<T, D, SMALL, false, false, false>(a, b, block, sequence(a, b), LaneSequences{}, Family{}, 0, kv_head, blockIdx.z, threadIdx.x, shared);
}

}  // namespace
}  // namespace ttmi
