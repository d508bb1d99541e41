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
struct Walk {  // 64 sequences, a lane each
  int base, rounds;       // number of the first; rounds of this lane's, for one head
  int64_t before, upto;   // units of all sequences before these; of these up to this lane's, it included
  int64_t groups;         // of batches of more than 64 sequences: units of this lane's 64th of them and of those before it
};
__device__ __forceinline__ int rounds_of(const PagedArgs& a, int b) {
  const Sequence seq = sequence(a, b);
  const int rows = seq.tokens * a.group;
  if (rows <= 0) return 0;
  if (rows > a.few) return a.every ? kStart + 1 : 0;  // (more rows than was said: not cut)
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
__device__ __forceinline__ void walk_to(const PagedArgs& a, Walk& w, int base, int64_t before) {
  const int lane = (int)(threadIdx.x % kWave);
  w.base = base, w.before = before;
  w.rounds = base + lane < a.view.batch ? rounds_of(a, base + lane) : 0;
  w.upto = sum_up_to_lane((int64_t)w.rounds * a.view.kv_heads);
}
__device__ __forceinline__ void walk_on(const PagedArgs& a, Walk& w) { walk_to(a, w, w.base + kWave, w.before + lane_of(w.upto, kWave - 1)); }
__device__ __forceinline__ int group_size(const PagedArgs& a) { return (a.view.batch + kWave - 1) / kWave; }
__device__ __forceinline__ void walk_to_group(const PagedArgs& a, Walk& w, int group) {
  walk_to(a, w, group * group_size(a), group > 0 ? lane_of(w.groups, group - 1) : 0);
}
// -> all units
__device__ __forceinline__ int64_t count_units(const PagedArgs& a, Walk& w) {
  w.groups = 0;
  if (a.view.batch <= kWave) {
    walk_to(a, w, 0, 0);
    return lane_of(w.upto, kWave - 1);
  }
  const int size = group_size(a), first = (int)(threadIdx.x % kWave) * size;
  int64_t mine = 0;
#pragma unroll 4
  for (int i = 0; i < size; ++i) mine += first + i < a.view.batch ? rounds_of(a, first + i) : 0;
  w.groups = sum_up_to_lane(mine * a.view.kv_heads);
  w.base = 0, w.rounds = 0, w.before = w.upto = 0;
  return lane_of(w.groups, kWave - 1);
}
struct Place {
  int b, kv_head, round, rounds;  // round: of this head's `rounds`
};
__device__ __forceinline__ Place find_unit(const PagedArgs& a, Walk& w, int64_t unit) {
  if (a.view.batch > kWave && (unit < w.before || unit >= w.before + lane_of(w.upto, kWave - 1)))
    walk_to_group(a, w, __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(w.groups > unit)) - 1));
  while (w.before + lane_of(w.upto, kWave - 1) <= unit) walk_on(a, w);
  const int64_t at = unit - w.before;
  const int found = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(w.upto > at)) - 1);
  Place p;
  p.b = w.base + found, p.rounds = __builtin_amdgcn_readlane(w.rounds, found);
  const int rest = (int)(at - (lane_of(w.upto, found) - (int64_t)p.rounds * a.view.kv_heads));
  p.kv_head = rest / p.rounds, p.round = rest - p.kv_head * p.rounds;
  return p;
}
// Workgroups that share the work.  At least kFewest rounds each, so that a wavefront has more than its first tile's wait.  us, 1 / 2 / 4 of them, 8 key heads of 128: 1 sequence
// of 1500 keys 11.6 / 12.5 / 15.6, of 8000 16.4 / 14.1 / 15.6, 8 of 1000 19.0 / 16.7 / 17.7, 8 of 2000 21.2 / 21.4 / 25.8.
constexpr int kFewest = 2;
__device__ __forceinline__ int64_t sharers(const PagedArgs& a, int64_t units) { return max((int64_t)1, min((int64_t)a.splits, (units + kFewest - 1) / kFewest)); }

// SMALL: pages of fewer than 16 slots
template <typename T, int D, int NW, bool SMALL>
__global__ __launch_bounds__(NW * 64, 8 / NW) void few_rows_kernel(const PagedArgs a) {
  using S = FewRows<T, D, NW>;
  __shared__ __align__(16) char smem[S::kLds];
  __shared__ float met[NW][kFewRows][2];
  const PagedView& view = a.view;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = lane & 15, quarter = lane >> 4;
  const T* const q = static_cast<const T*>(a.q);
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  char* const tile = smem + wave * S::kValueBytes;

  // splits 0: a workgroup for each pair
  Walk walk;
  int64_t unit = blockIdx.x, stop = unit + 1;
  if (a.splits > 0) {
    const int64_t units = count_units(a, walk), workgroups = sharers(a, units);
    if (blockIdx.x >= workgroups) return;
    unit = units * blockIdx.x / workgroups, stop = units * (blockIdx.x + 1) / workgroups;
  }
  while (unit < stop) {
    Place place;
    if (a.splits > 0) place = find_unit(a, walk, unit);
    else place.b = (int)(unit / view.kv_heads), place.kv_head = (int)(unit % view.kv_heads), place.round = 0, place.rounds = INT32_MAX;
    const int b = place.b, kv_head = place.kv_head;
    const int64_t ends = a.splits > 0 ? min(stop, unit + place.rounds - place.round) : stop;
    const int start = a.splits > 0 ? kStart : 0;  // (in a pair's first unit there is nothing to do)
    const int round0 = max(0, place.round - start), round1 = place.round + (int)(a.splits > 0 ? ends - unit : INT32_MAX) - start;
    const bool complete = round0 == 0 && round1 == place.rounds - start;
    unit = ends;
    if (round1 <= round0) continue;
    const Sequence seq = sequence(a, b);
    const int rows_all = seq.tokens * a.group;
    if (rows_all <= 0 || (rows_all > a.few && !a.every)) return;  // (a workgroup of its own)
    if (round0 == 0 && kv_head == 0 && tid == 0 && view.lengths[b] > seq.length) page_error(view);
    PageCursor cursor;
    cursor.table = view.table + (int64_t)b * view.table_pitch;
    cursor.first = 0, cursor.ahead = 0, cursor.at = 0;

    for (int row0 = 0; row0 < rows_all; row0 += kFewRows) {
      const int rows = min(kFewRows, rows_all - row0);
      const int token0 = row0 / a.group, token1 = (row0 + rows - 1) / a.group;
      const int token = row < rows ? (row0 + row) / a.group : token0, head = kv_head * a.group + (row < rows ? row0 + row - token * a.group : 0);
      const Reach mine = seq.reach(a, token), low = seq.reach(a, token0), high = seq.reach(a, token1);
      // Keys that some row sees, and those that all rows see: both ends rise with the position.  (A row without keys, before the first one, begins and ends at 0.)
      const int first = low.begin, end = max(low.end, high.end), sure_first = high.begin, sure_end = low.end;
      int lo = first & ~(S::kKeys - 1), hi = end;
      if (!complete) {
        lo = max(lo, (first / kRound + round0) * kRound);
        hi = min(hi, (first / kRound + round1) * kRound);
      }
      cursor.last = max(0, (end - 1) >> view.page_shift);

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
      auto work_on = [&](int key, auto more) __attribute__((always_inline)) {
        const bool masked = key < sure_first || key + S::kKeys > sure_end || key + S::kKeys > hi;
        uint32_t wild = 0;
        if (masked) {  // keys that no row sees may hold anything: their values count as zeros, and one that only some rows see must not reach the others
  #pragma unroll
          for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
            for (int i = 0; i < S::kValuePieces; ++i) {
              const int k = key + 16 * g + (i * 1024 + lane * 16) / S::kRowBytes;
              if (k < first || k >= end) vf[g][i] = u32x4{0u, 0u, 0u, 0u};
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
        if constexpr (decltype(more)::value) load_values(key + kStep);

        floatx4 st[S::kGroups];
  #pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          st[g] = floatx4{0.f, 0.f, 0.f, 0.f};
  #pragma unroll
          for (int i = 0; i < S::kSteps; ++i) st[g] = mma16<T>(kf[g][i], qf[i], st[g]);
        }
        if constexpr (decltype(more)::value) load_keys(key + kStep);
        if (masked) {
  #pragma unroll
          for (int g = 0; g < S::kGroups; ++g)
  #pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = key + 16 * g + 4 * quarter + e;
              if (k < mine.begin || k >= mine.end || k >= hi) st[g][e] = -INFINITY;
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
          for (int k = key; k < min(key + S::kKeys, hi); ++k) {
            const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * quarter;
            const bool seen = k >= mine.begin && k < mine.end;
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
      int key = lo + wave * S::kKeys;
      if (key < hi) {
        if constexpr (!SMALL) fetch_pages<S::kRowBytes>(view, cursor, kv_head, key);
        load_values(key);
        load_keys(key);
        for (; key + kStep < hi; key += kStep) work_on(key, std::true_type{});
        work_on(key, std::false_type{});
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
          if (complete) {
            const int t = (row0 + r) / a.group, h = kv_head * a.group + row0 + r - t * a.group;
            const float inv = inverse_sum(total, seq.reach(a, t).end > 0);
            T* to = static_cast<T*>(a.out) + (seq.start + t) * a.out_pitch + (int64_t)h * D + d0;
            Vec<T, kWide> x;
  #pragma unroll
            for (int c = 0; c < kWide; ++c) x.v[c] = from_float<T>(o[c] * inv);
            store_vec<T, kWide>(to, x);
          } else {
            const int64_t at = (2 * (int64_t)blockIdx.x + (round0 == 0 ? 1 : 0)) * kFewRows + r;
            float* const ml = a.partial + 2 * (int64_t)a.splits * kFewRows * D + at * 2;
  #pragma unroll
            for (int c = 0; c < kWide; ++c) a.partial[at * D + d0 + c] = o[c];
            if (d0 == 0) ml[0] = best, ml[1] = total;
          }
        }
      }
      if (row0 + kFewRows < rows_all || unit < stop) __syncthreads();
    }
  }
}

// Pairs that were several workgroups': their rows' partial results are joined, in 5 to 7 us, nearly all of them the launch and three trips to memory.  A workgroup per pair and row, or per pair where there are many of them: then a wavefront
// takes a row.
// us, a workgroup per row / per pair, 32 query and 8 key heads of 128: 1 sequence of 3000 keys 12.8 / 14.2, 8 (64 pairs) 24.9 / 25.4, 64 of 1500 (512) 75.4 / 73.8, 200 (1600)
// 241 / 228; 16 query heads of one key head, one sequence of 100000 keys beside 63 of 500, whose pair has most of the parts, 45.7 / 145.
constexpr int kManyPairs = 512;
template <typename T, int D>
__global__ __launch_bounds__(256) void join_few_rows_kernel(const PagedArgs a, bool by_pair) {
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, b = blockIdx.x / view.kv_heads;
  const Sequence seq = sequence(a, b);
  const int rows = seq.tokens * a.group;
  if (rows > a.few || (int)blockIdx.y >= rows) return;
  Walk walk;
  const int64_t units = count_units(a, walk), workgroups = sharers(a, units);
  if (view.batch > kWave) walk_to_group(a, walk, b / group_size(a));
  while (walk.base + kWave <= b) walk_on(a, walk);
  const int lane = b - walk.base, rounds = __builtin_amdgcn_readlane(walk.rounds, lane);
  const int64_t unit = walk.before + lane_of(walk.upto, lane) - (int64_t)rounds * (view.kv_heads - kv_head);
  const int64_t first = ((unit + kStart + 1) * workgroups - 1) / units, last = ((unit + rounds) * workgroups - 1) / units;
  if (first == last) return;
  const int parts = (int)(last - first) + 1;
  const float* const ml = a.partial + 2 * (int64_t)a.splits * kFewRows * D;
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

}  // namespace

int launch_few_rows(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream) {
  const unsigned pairs = (unsigned)((int64_t)a.view.batch * a.view.kv_heads);
  const bool by_pair = pairs >= kManyPairs;
  TTMI_DISPATCH_FLOAT(dtype, T, {
    auto launch = [&](auto kernel, auto join) {
      hipLaunchKernelGGL(kernel, dim3(a.splits > 0 ? (unsigned)a.splits : pairs), dim3(a.waves * 64), 0, stream, a);
      if (a.splits > 0) hipLaunchKernelGGL(join, dim3(pairs, by_pair ? 1u : (unsigned)std::min<int64_t>(a.few, (int64_t)a.view.tokens * a.group)), dim3(256), 0, stream, a, by_pair);
    };
    const bool small = a.view.page_shift < 4;
    auto sized = [&](auto d) {
      constexpr int D = decltype(d)::value;
      if (small && a.waves == 4) launch(few_rows_kernel<T, D, 4, true>, join_few_rows_kernel<T, D>);
      else if (small) launch(few_rows_kernel<T, D, 8, true>, join_few_rows_kernel<T, D>);
      else if (a.waves == 4) launch(few_rows_kernel<T, D, 4, false>, join_few_rows_kernel<T, D>);
      else launch(few_rows_kernel<T, D, 8, false>, join_few_rows_kernel<T, D>);
    };
    if (head_dim == 64) sized(std::integral_constant<int, 64>{});
    else sized(std::integral_constant<int, 128>{});
  });
  return launch_status("paged_attention");
}

}  // namespace ttmi
