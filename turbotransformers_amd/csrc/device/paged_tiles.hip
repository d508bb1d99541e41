// Attention over pages where sequences have many rows (new tokens times query heads of a key/value head): prompts and chunks of them.
//
// The matrix instructions bound it, and with them the exponentials and what LDS can feed.  A workgroup has 128 rows of one sequence and head, 32 a wavefront, and
// walks over tiles of 64 keys (fp32: 32) that all four share in LDS, fetched into registers one ahead and stored while the other stage is worked on.
// Scores are computed transposed, St[key, row] = K . Q^T (v_mfma_f32_32x32x16, fp32: 32x32x2), so a lane has one row, its statistics need one exchange of the two
// half-wavefronts, and the probabilities lie in the accumulators as Ot[d, row] += Vt . Pt wants them; Vt is what the transposing reads give of values that lie in LDS
// row by row as in the cache (fp32: plain reads of a column).  Packing a group's heads into one tile of rows reads the keys of a head once for all of them and keeps
// tiles full whatever the group.
#include "paged_attention.h"

namespace ttmi {
namespace {

constexpr int kTileRows = 128;  // of a workgroup

template <typename T, int D>
struct Tiles {
  static constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;
  static constexpr int kSubs = kKeys / 32;
  static constexpr int kElems = 16 / (int)sizeof(T);
  static constexpr int kRowBytes = D * (int)sizeof(T);
  static constexpr int kBytes = kKeys * kRowBytes;      // of a tile of keys, or of values
  static constexpr int kPieces = kBytes / 4096;         // 16-byte pieces of a tile per thread
  static constexpr int kSteps = kRowBytes / 32;         // pieces of a row per lane, for the first product
  static constexpr int kOut = D / 32;
};

// Places of a row's 16-byte pieces in LDS.  Keys: sixteen rows read the same piece at a time.  Values: 64 bytes of four rows at a time (fp32: 128 bytes of two rows that lie
// four apart).  The exclusive or takes them to different banks.
template <typename T, int D>
__device__ __forceinline__ int key_piece(int row, int piece) {
  if constexpr (sizeof(T) == 2 && D == 64) return piece ^ ((row >> 1) & 7);
  else return piece ^ (row & 15);
}
template <typename T, int D>
__device__ __forceinline__ int value_piece(int row, int piece) {
  if constexpr (sizeof(T) == 4) return piece ^ (((row >> 2) & 1) << 3);
  else if constexpr (D == 128) return piece ^ ((row & 3) << 2);
  else return piece ^ (((row >> 1) & 1) << 2);
}

// A row's sums over one part of its keys: divided and stored, or, where its keys lie in several parts, kept for the kernel that joins those.
template <typename T, int D>
__device__ __forceinline__ void store_rows(const PagedArgs& a, const Sequence& seq, int token, int head, int part, int part0, int part1, int lhalf,
                                           const floatx16 (&ot)[D / 32], float top, float sum) {
  const int64_t at_token = seq.start + token;
  if (part0 == part1) {
    if (part != part0) return;
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    T* to = static_cast<T*>(a.out) + at_token * a.out_pitch + (int64_t)head * D + 4 * lhalf;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        Vec<T, 4> x;
#pragma unroll
        for (int c = 0; c < 4; ++c) x.v[c] = from_float<T>(ot[t][4 * g + c] * inv);
        store_vec<T, 4>(to + 32 * t + 8 * g, x);
      }
    return;
  }
  const int64_t at = (at_token * a.heads + head) * a.splits + part;
  float* to = a.partial + at * D + 4 * lhalf;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<floatx4*>(to + 32 * t + 8 * g) = floatx4{ot[t][4 * g], ot[t][4 * g + 1], ot[t][4 * g + 2], ot[t][4 * g + 3]};
  if (lhalf == 0) {
    float* ml = a.partial + (int64_t)a.view.tokens * a.heads * a.splits * D + at * 2;
    ml[0] = top, ml[1] = sum;
  }
}

// The `want`-th block of rows of all sequences -> its sequence and number in it (false: there are fewer).  Every lane looks at a sequence.
template <int ROWS>
__device__ __forceinline__ bool find_block(const PagedArgs& a, int want, int* b, int* block) {
  const int lane = (int)(threadIdx.x % kWave);
  for (int base = 0; base < a.view.batch; base += kWave) {
    int blocks = 0;
    if (base + lane < a.view.batch) {
      const int rows = sequence(a, base + lane).tokens * a.group;
      if (rows > kFewRows || a.every) blocks = (rows + ROWS - 1) / ROWS;
    }
    int upto = blocks;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int below = __shfl_up(upto, d, kWave);
      if (lane >= d) upto += below;
    }
    const uint64_t past = __ballot(upto > want);
    if (past != 0) {
      const int found = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)past) - 1);
      *b = base + found;
      // the last rows have the most keys before them: they begin first
      *block = __builtin_amdgcn_readlane(upto, found) - 1 - want;
      return true;
    }
    want -= __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

// SMALL: pages of fewer than 16 slots
template <typename T, int D, bool SMALL>
__global__ __launch_bounds__(256, 2) void tiles_kernel(const PagedArgs a) {
  using S = Tiles<T, D>;
  __shared__ __align__(16) char smem[4 * S::kBytes];
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, part = blockIdx.z;
  int b, block;
  if (!find_block<kTileRows>(a, blockIdx.x / view.kv_heads, &b, &block)) return;
  const Sequence seq = sequence(a, b);
  const int chunk = seq.chunk(a);
  const int row0 = block * kTileRows, rows = min(kTileRows, seq.tokens * a.group - row0);
  if (part == 0 && kv_head == 0 && block == 0 && threadIdx.x == 0 && view.lengths[b] > seq.length) page_error(view);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lrow = lane & 31, lhalf = lane >> 5;
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  // keys that some row of the workgroup sees, and those that all see (both ends rise with the position); the same of this wavefront
  const Reach low = seq.reach(a, row0 / a.group), high = seq.reach(a, (row0 + rows - 1) / a.group);
  const int first = low.begin, end = max(low.end, high.end), sure_first = high.begin, sure_end = low.end;
  const int lo = (int)max(part * (int64_t)chunk, (int64_t)(first & ~(S::kKeys - 1))), hi = (int)min((part + 1) * (int64_t)chunk, (int64_t)end);
  if (lo >= hi && part != 0) return;
  const int wave_rows = max(0, min(32, rows - wave * 32));
  const int wrow = row0 + wave * 32;
  const Reach wave_low = seq.reach(a, wrow / a.group), wave_high = seq.reach(a, (wrow + max(wave_rows, 1) - 1) / a.group);
  const int wave_first = wave_low.begin, wave_end = wave_rows > 0 ? max(wave_low.end, wave_high.end) : 0;
  const bool live = lrow < wave_rows;
  const int token = (wrow + (live ? lrow : 0)) / a.group, head = kv_head * a.group + (live ? wrow + lrow - token * a.group : 0);
  const Reach mine = seq.reach(a, token);

  u32x4 qf[S::kSteps];
#pragma unroll
  for (int i = 0; i < S::kSteps; ++i) {
    qf[i] = u32x4{0u, 0u, 0u, 0u};
    if (live) qf[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + (seq.start + token) * a.q_pitch + (int64_t)head * D + (2 * i + lhalf) * S::kElems);
  }
  floatx16 ot[S::kOut];
#pragma unroll
  for (int t = 0; t < S::kOut; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) ot[t][e] = 0.f;
  float top = -INFINITY, sum = 0.f;

  PageCursor cursor;
  cursor.table = view.table + (int64_t)b * view.table_pitch;
  cursor.last = max(0, (end - 1) >> view.page_shift);
  cursor.first = 0, cursor.ahead = 0, cursor.at = 0;
  u32x4 kr[S::kPieces], vr[S::kPieces];
  // 16-byte pieces of a tile: thread by thread, 4 KB after 4 KB.  A wavefront's 1 KB lies in one group of 16 rows.
  auto load_piece = [&](int i, int key) __attribute__((always_inline)) {
    if constexpr (!SMALL) {
      if (i == 0) come_to<S::kRowBytes>(view, cursor, kv_head, key);
      const int group = (i * 4096 + wave * 1024) / (16 * S::kRowBytes) * 16;
      const int64_t from = group_at<S::kRowBytes>(view, cursor, key + group);
      const uint32_t in_group = (uint32_t)(i * 4096 + tid * 16) % (16 * S::kRowBytes);
      kr[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(keys) + from + in_group);
      vr[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(values) + from + in_group);
    } else {
      const int at = i * 4096 + tid * 16;
      const int64_t from = row_offset<D>(view, cursor, kv_head, key + at / S::kRowBytes) + at % S::kRowBytes / (int)sizeof(T);
      kr[i] = *reinterpret_cast<const u32x4*>(keys + from);
      vr[i] = *reinterpret_cast<const u32x4*>(values + from);
    }
  };
  auto key_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * S::kBytes; };
  auto value_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * S::kBytes + S::kBytes; };
  auto store_piece = [&](int i, int s) __attribute__((always_inline)) {
    const int at = i * 4096 + tid * 16, r = at / S::kRowBytes, c = at % S::kRowBytes / 16;
    *reinterpret_cast<u32x4*>(key_stage(s) + r * S::kRowBytes + key_piece<T, D>(r, c) * 16) = kr[i];
    *reinterpret_cast<u32x4*>(value_stage(s) + r * S::kRowBytes + value_piece<T, D>(r, c) * 16) = vr[i];
  };
  // Keys that no row sees may hold anything: their values count as zeros.  Where only some rows see a key, infinities and NaNs of its values must not
  // reach the others: they are left out here (-> whether there are any) and added where they are seen.
  auto partly_seen = [&](int key) __attribute__((always_inline)) { return key < sure_first || key + S::kKeys > sure_end; };
  auto clean_values = [&](int key) __attribute__((always_inline)) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int k = key + (i * 4096 + tid * 16) / S::kRowBytes;
      if (k < first || k >= end) vr[i] = u32x4{0u, 0u, 0u, 0u};
      found |= not_finite<T>(vr[i]);
      vr[i] = finite_part<T>(vr[i]);
    }
    return found;
  };
  auto barrier = [&](bool partly, uint32_t found) __attribute__((always_inline)) -> bool {
    if (partly) return __syncthreads_or((int)found) != 0;
    __syncthreads();
    return false;
  };

  if (lo < hi) {
    // (Loads past the last tile fetch that once more, out of L2: a load that may or may not have been sent would make the compiler wait for all of them.)
    const int last = lo + (hi - 1 - lo) / S::kKeys * S::kKeys;
    if constexpr (!SMALL) fetch_pages<S::kRowBytes>(view, cursor, kv_head, lo);
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) load_piece(i, lo);
    uint32_t found = partly_seen(lo) ? clean_values(lo) : 0;
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) store_piece(i, 0);
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) load_piece(i, min(lo + S::kKeys, last));
    bool wild = barrier(partly_seen(lo), found);
    // One tile; its stage is known to the compiler, so that places in LDS are fixed numbers behind one of the lane's.
    auto work_on = [&](int key, auto stage) __attribute__((always_inline)) {
      constexpr int s = decltype(stage)::value;
      // The other stage is free: what was fetched for it while the last tile was worked on goes there, and the tile behind it is sent for.
      const bool next_partly = partly_seen(key + S::kKeys);
      const int after = min(key + 2 * S::kKeys, last);
      found = next_partly ? clean_values(key + S::kKeys) : 0;
      if (key >= wave_end || key + S::kKeys <= wave_first) {  // nothing to do for this wavefront's rows
#pragma unroll
        for (int i = 0; i < S::kPieces; ++i) store_piece(i, s ^ 1);
#pragma unroll
        for (int i = 0; i < S::kPieces; ++i) load_piece(i, after);
        wild = barrier(next_partly, found);
        return;
      }
      const char* const kt = key_stage(s);
      const char* const vt = value_stage(s);
      floatx16 st[S::kSubs];
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) st[u][e] = 0.f;
      auto read_keys = [&](int n) __attribute__((always_inline)) {  // the operand of the n-th matrix instruction of St
        const int r = 32 * (n % S::kSubs) + lrow;
        return *reinterpret_cast<const u32x4*>(kt + r * S::kRowBytes + key_piece<T, D>(r, 2 * (n / S::kSubs) + lhalf) * 16);
      };
      // Reads run kAhead instructions before their use.  The fences keep that order: left to itself the compiler waits for each read in front of its use.
      constexpr int kAhead = 4, kScores = S::kSubs * S::kSteps;
      u32x4 f[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) f[n] = read_keys(n);
#pragma unroll
      for (int n = 0; n < kScores; ++n) {
        st[n % S::kSubs] = mma32<T>(f[n % kAhead], qf[n / S::kSubs], st[n % S::kSubs]);
        if (n + kAhead < kScores) f[n % kAhead] = read_keys(n + kAhead);
        if (n < S::kPieces) store_piece(n, s ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < S::kPieces; ++i) load_piece(i, after);
      if (key < wave_high.begin || key + S::kKeys > wave_low.end) {
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int k = key + 32 * u + 8 * (e / 4) + 4 * lhalf + e % 4;
            if (k < mine.begin || k >= mine.end) st[u][e] = -INFINITY;
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
      if (__any(shrink != 1.f)) {
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
            const u32x2 half = read_transposed(vt + r * S::kRowBytes + value_piece<T, D>(r, 4 * t + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8);
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
      } else {
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            st[u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[u][e], a.scale_log2e, -zero));
            sum += st[u][e];
            const int r = 32 * u + 8 * (e / 4) + 4 * lhalf + e % 4;
#pragma unroll
            for (int t = 0; t < S::kOut; ++t) {
              const float v = *reinterpret_cast<const float*>(vt + r * S::kRowBytes + value_piece<T, D>(r, 8 * t + (lrow >> 2)) * 16 + (lrow & 3) * 4);
              ot[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, st[u][e], ot[t], 0, 0, 0);
            }
          }
      }
      if (wild) {  // an infinity or a NaN is what a sum with it is, whatever its weight
#pragma unroll 1
        for (int k = key; k < min(key + S::kKeys, hi); ++k) {
          const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * lhalf;
          const bool seen = k >= mine.begin && k < mine.end;
#pragma unroll
          for (int t = 0; t < S::kOut; ++t) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const T x = v[32 * t + 8 * (e / 4) + e % 4];
              if (seen && wild_value(x)) ot[t][e] += to_float(x);
            }
            __builtin_amdgcn_sched_barrier(0);  // (few registers: this path is cold)
          }
        }
      }
      wild = barrier(next_partly, found);
    };
    for (int key = lo; key < hi; key += 2 * S::kKeys) {
      work_on(key, std::integral_constant<int, 0>{});
      if (key + S::kKeys < hi) work_on(key + S::kKeys, std::integral_constant<int, 1>{});
    }
  }

  {
    const LanePair both = swap_halves(sum);
    sum = both.a + both.b;
  }
  if (!live) return;
  store_rows<T, D>(a, seq, token, head, part, mine.begin / chunk, mine.end > 0 ? (mine.end - 1) / chunk : 0, lhalf, ot, top, sum);
}

// The 16-bit types.  A workgroup has 256 rows, 32 for each of its eight wavefronts (two on a SIMD), and goes through the keys 32 at a time.  At a step j the matrix
// instructions of the scores of step j + 1 and of the output of step j - 1 run beside the exponentials of step j, which they do not wait for; order is kept by scheduling
// fences, since the compiler by itself puts every read of LDS in front of its use.
constexpr int kStepRows = 256;

template <typename T, int D>
struct Steps {
  static constexpr int kKeys = 32;
  static constexpr int kElems = 8;                  // of a 16-byte piece
  static constexpr int kRowBytes = D * 2;
  static constexpr int kBytes = kKeys * kRowBytes;  // of the keys of a step, or of its values
  static constexpr int kScores = D / 16;            // matrix instructions of a step's scores
  static constexpr int kOut = D / 32;
  static constexpr int kProducts = 2 * kOut;        // of its part of the output
  static constexpr bool kBoth = kBytes / 16 >= 512; // every thread fetches a piece of the keys and one of the values; else one half of the workgroup fetches each
};

template <typename T, int D, bool SMALL>
__global__ __launch_bounds__(512, 2) void steps_kernel(const PagedArgs a) {
  using S = Steps<T, D>;
  __shared__ __align__(16) char smem[4 * S::kBytes];
  __shared__ int wild;  // whether values that only some rows see hold infinities or NaNs
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, part = blockIdx.z;
  int b, block;
  if (!find_block<kStepRows>(a, blockIdx.x / view.kv_heads, &b, &block)) return;
  const Sequence seq = sequence(a, b);
  const int chunk = seq.chunk(a);
  const int row0 = block * kStepRows, rows = min(kStepRows, seq.tokens * a.group - row0);
  if (part == 0 && kv_head == 0 && block == 0 && threadIdx.x == 0 && view.lengths[b] > seq.length) page_error(view);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lrow = lane & 31, lhalf = lane >> 5;
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  // keys that some row of the workgroup sees, and those that all see (both ends rise with the position); the same of this wavefront
  const Reach low = seq.reach(a, row0 / a.group), high = seq.reach(a, (row0 + rows - 1) / a.group);
  const int first = low.begin, end = max(low.end, high.end);
  const int lo = (int)max(part * (int64_t)chunk, (int64_t)(first & ~(S::kKeys - 1))), hi = (int)min((part + 1) * (int64_t)chunk, (int64_t)end);
  if (lo >= hi && part != 0) return;
  const int sure_first = high.begin, sure_end = min(low.end, hi);
  const int wrow = row0 + wave * 32, wave_rows = max(0, min(32, rows - wave * 32));
  const bool active = wave_rows > 0;
  const Reach wave_low = seq.reach(a, (active ? wrow : row0) / a.group), wave_high = seq.reach(a, (active ? wrow + wave_rows - 1 : row0) / a.group);
  const bool live = lrow < wave_rows;
  const int token = (live ? wrow + lrow : row0) / a.group, head = kv_head * a.group + (live ? wrow + lrow - token * a.group : 0);
  Reach mine = seq.reach(a, token);
  const int part0 = mine.begin / chunk, part1 = mine.end > 0 ? (mine.end - 1) / chunk : 0;

  u32x4 qf[S::kScores];
#pragma unroll
  for (int i = 0; i < S::kScores; ++i) {
    qf[i] = u32x4{0u, 0u, 0u, 0u};
    if (live) qf[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + (seq.start + token) * a.q_pitch + (int64_t)head * D + (2 * i + lhalf) * S::kElems);
  }
  floatx16 ot[S::kOut], st[2];
#pragma unroll
  for (int t = 0; t < S::kOut; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) ot[t][e] = 0.f;
  float top = -INFINITY, sum = 0.f;

  if (lo < hi) {
    const int steps = (hi - lo + S::kKeys - 1) / S::kKeys;
    mine.end = min(mine.end, hi);  // (of this part)
    const int wave_first = wave_high.begin, wave_end = min(wave_low.end, hi);
    if (tid == 0) wild = 0;
    // This thread's pieces of a step: where they come from and where in LDS they go.
    const int at = (S::kBoth ? tid : tid & 255) * 16, piece_row = at / S::kRowBytes;
    const int group = (S::kBoth ? wave : wave & 3) * 1024 / (16 * S::kRowBytes) * 16;
    const uint32_t in_group = (uint32_t)at % (16 * S::kRowBytes);
    const bool fetches_keys = S::kBoth || wave < 4, fetches_values = S::kBoth || wave >= 4;
    char* const key_place = smem + piece_row * S::kRowBytes + key_piece<T, D>(piece_row, at % S::kRowBytes / 16) * 16;
    char* const value_place = smem + 2 * S::kBytes + piece_row * S::kRowBytes + value_piece<T, D>(piece_row, at % S::kRowBytes / 16) * 16;
    PageCursor key_cursor, value_cursor;
    key_cursor.table = value_cursor.table = view.table + (int64_t)b * view.table_pitch;
    key_cursor.last = value_cursor.last = max(0, (end - 1) >> view.page_shift);
    if constexpr (!SMALL) {
      fetch_pages<S::kRowBytes>(view, key_cursor, kv_head, lo);
      value_cursor = key_cursor;
    }
    // (Steps past the last one fetch that again, out of L2: a load that may or may not have been sent would make the compiler wait for all of them.)
    auto fetch = [&](const T* from, PageCursor& cursor, int step) __attribute__((always_inline)) {
      const int key = lo + min(step, steps - 1) * S::kKeys;
      if constexpr (SMALL) {
        return *reinterpret_cast<const u32x4*>(from + row_offset<D>(view, cursor, kv_head, key + piece_row) + at % S::kRowBytes / 2);
      } else {
        return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(from) + group_at<S::kRowBytes>(view, cursor, key + group) + in_group);
      }
    };
    // What is fetched at step j is stored at step j + 2: the keys of step j + 4, which are read at step j + 3, and the values of step j + 2, read at step j + 3.
    u32x4 kr[2], vr[2];
    auto store_keys = [&](const u32x4& x, int stage) __attribute__((always_inline)) {
      if (fetches_keys) *reinterpret_cast<u32x4*>(key_place + stage * S::kBytes) = x;
    };
    auto store_values = [&](const u32x4& x, int stage) __attribute__((always_inline)) {
      if (fetches_values) *reinterpret_cast<u32x4*>(value_place + stage * S::kBytes) = x;
    };
    auto fetch_both = [&](int j, int parity) __attribute__((always_inline)) {
      if constexpr (S::kBoth) {
        kr[parity] = fetch(keys, key_cursor, j + 4);
        vr[parity] = fetch(values, value_cursor, j + 2);
      } else {
        kr[parity] = vr[parity] = fetch(fetches_keys ? keys : values, key_cursor, fetches_keys ? j + 4 : j + 2);
      }
    };
    // The pages of what steps j and j + 1 fetch (j even: both are in the same 64 pages).  Not in the middle of a step, which is to be one piece of straight code.
    auto turn_pages = [&](int j) __attribute__((always_inline)) {
      if constexpr (!SMALL) {
        auto key_of = [&](int step) { return lo + min(step, steps - 1) * S::kKeys; };
        come_to<S::kRowBytes>(view, key_cursor, kv_head, key_of(S::kBoth || fetches_keys ? j + 4 : j + 2));
        if constexpr (S::kBoth) come_to<S::kRowBytes>(view, value_cursor, kv_head, key_of(j + 2));
      }
    };
    // the n-th operand of a step's scores, and of its output
    auto read_keys = [&](int n, int stage) __attribute__((always_inline)) {
      return *reinterpret_cast<const u32x4*>(smem + stage * S::kBytes + lrow * S::kRowBytes + key_piece<T, D>(lrow, 2 * n + lhalf) * 16);
    };
    auto read_values = [&](int n, int stage) __attribute__((always_inline)) {
      const int t = n % S::kOut;
      u32x4 v;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int r = 16 * (n / S::kOut) + 8 * g + 4 * lhalf + ((lane >> 2) & 3);
        const u32x2 half = read_transposed(smem + (2 + stage) * S::kBytes + r * S::kRowBytes +
                                           value_piece<T, D>(r, 4 * t + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8);
        v[2 * g] = half[0], v[2 * g + 1] = half[1];
      }
      return v;
    };
    auto partly_seen = [&](int key) __attribute__((always_inline)) { return key < sure_first || key + S::kKeys > sure_end; };
    // An infinity or a NaN among values that only some rows see is what a sum with it is, whatever its weight.
    auto add_wild = [&](int key) __attribute__((always_inline)) {
#pragma unroll 1
      for (int k = key; k < min(key + S::kKeys, hi); ++k) {
        const T* v = values + row_offset<D>(view, key_cursor, kv_head, k) + 4 * lhalf;
        const bool seen = k >= mine.begin && k < mine.end;
#pragma unroll
        for (int t = 0; t < S::kOut; ++t) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const T x = v[32 * t + 8 * (e / 4) + e % 4];
            if (seen && wild_value(x)) ot[t][e] += to_float(x);
          }
          __builtin_amdgcn_sched_barrier(0);  // (few registers: this path is cold)
        }
      }
    };

    // The first two steps' keys go to their stages, the two behind them and the first two steps' values are on their way.  There are no values before the first step's.
    {
      const u32x4 k0 = fetch(keys, key_cursor, 0), k1 = fetch(keys, key_cursor, 1);
      fetch_both(-2, 0);
      fetch_both(-1, 1);
      store_keys(k0, 0);
      store_keys(k1, 1);
      store_values(u32x4{0u, 0u, 0u, 0u}, 1);
    }
    __syncthreads();
    // Keys that no row sees may hold anything: their values count as zeros.  Infinities and NaNs of values that only some rows see must not reach the others: they are
    // left out and noted.
    auto settle = [&](u32x4& x, int key) __attribute__((always_inline)) {
      const int k = key + piece_row;
      if (k < first || k >= hi) x = u32x4{0u, 0u, 0u, 0u};
      if (fetches_values && not_finite<T>(x)) wild = 1;
      x = finite_part<T>(x);
    };
    if (!active) {  // no rows: this wavefront only fetches
      __syncthreads();
      for (int j = 0; j < steps; j += 2) {
        turn_pages(j);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          if (partly_seen(lo + (j + p) * S::kKeys)) settle(vr[p], lo + (j + p) * S::kKeys);
          store_keys(kr[p], p);
          store_values(vr[p], p);
          fetch_both(j + p, p);
          __syncthreads();
        }
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) st[0][e] = 0.f;
#pragma unroll
    for (int n = 0; n < S::kScores; ++n) st[0] = mma32<T>(read_keys(n, 0), qf[n], st[0]);
    __syncthreads();

    u32x4 pf[2][2] = {};  // probabilities of a step, rounded to the type, as the operands of its output
    constexpr int kAhead = 4, kAll = S::kProducts + S::kScores;
    auto work_on = [&](int j, auto parity) __attribute__((always_inline)) {
      constexpr int P = decltype(parity)::value, N = P ^ 1;
      const int key = lo + j * S::kKeys;
      if (__builtin_expect(partly_seen(key), 0)) settle(vr[P], key);
      auto operand = [&](int n) __attribute__((always_inline)) { return n < S::kProducts ? read_values(n, N) : read_keys(n - S::kProducts, N); };
      u32x4 f[kAhead];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) f[n] = operand(n);
      __builtin_amdgcn_sched_barrier(0);
      floatx16& s = st[P];
      if (__builtin_expect(key < wave_first || key + S::kKeys > wave_end, 0)) {
        const int from = mine.begin - key - 4 * lhalf;
        const uint32_t span = (uint32_t)max(0, mine.end - mine.begin);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((uint32_t)(8 * (e / 4) + e % 4 - from) >= span) s[e] = -INFINITY;
      }
      float zero;
      {
        float m[4];  // (chains of a quarter of the length)
#pragma unroll
        for (int c = 0; c < 4; ++c) m[c] = fmaxf(fmaxf(s[c], s[c + 4]), fmaxf(s[c + 8], s[c + 12]));
        const LanePair sw = swap_halves(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
        const float moved = moved_reference(top, fmaxf(sw.a, sw.b) * a.scale_log2e);
        zero = moved == -INFINITY ? 0.f : moved;  // (a row that has seen no key yet)
        if (__builtin_expect(__any(moved != top), 0)) {
          // references are whole numbers, so this is a power of two and the rounded probabilities of the step before take it exactly
          const float shrink = __builtin_amdgcn_exp2f(top - zero);
          sum *= shrink;
#pragma unroll
          for (int t = 0; t < S::kOut; ++t) ot[t] *= shrink;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) pf[N][i][w] = scale_pair<T>(pf[N][i][w], shrink);
          top = moved;
        }
      }
      auto probabilities = [&](int pair) __attribute__((always_inline)) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * pair], a.scale_log2e, -zero));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * pair + 1], a.scale_log2e, -zero));
        pf[P][pair / 4][pair % 4] = pack2<T>(p0, p1);
        // the sum is that of the rounded ones, so what rounding does to all of them alike cancels
        sum = add_pair<T>(pf[P][pair / 4][pair % 4], sum);
        asm volatile("" : "+v"(sum));  // (here, not where the next step wants it)
      };
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < kAll; ++n) {
        if (n < S::kProducts) ot[n % S::kOut] = mma32<T>(f[n % kAhead], pf[N][n / S::kOut], ot[n % S::kOut]);
        else if (n == S::kProducts) st[N] = mma32<T>(f[n % kAhead], qf[0], floatx16{});
        else st[N] = mma32<T>(f[n % kAhead], qf[n - S::kProducts], st[N]);
        if (n + kAhead < kAll) f[n % kAhead] = operand(n + kAhead);
        if (n == 1) store_keys(kr[P], P);
        if (n == 2) store_values(vr[P], P);
        if (n == 3) fetch_both(j, P);
#pragma unroll
        for (int i = n * 8 / kAll; i < (n + 1) * 8 / kAll; ++i) probabilities(i);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (__builtin_expect(partly_seen(key - S::kKeys), 0) && j > 0 && wild) add_wild(key - S::kKeys);
      __syncthreads();
    };
    // (An odd number of steps has one more of keys that no row sees.)
    for (int j = 0; j < steps; j += 2) {
      turn_pages(j);
      work_on(j, std::integral_constant<int, 0>{});
      work_on(j + 1, std::integral_constant<int, 1>{});
    }
    // the last step's part of the output
    const int key = lo + ((steps - 1) | 1) * S::kKeys;
#pragma unroll
    for (int n = 0; n < S::kProducts; ++n) ot[n % S::kOut] = mma32<T>(read_values(n, 1), pf[1][n / S::kOut], ot[n % S::kOut]);
    if (partly_seen(key) && wild) add_wild(key);
  }

  {
    const LanePair both = swap_halves(sum);
    sum = both.a + both.b;
  }
  if (live) store_rows<T, D>(a, seq, token, head, part, part0, part1, lhalf, ot, top, sum);
}

// Rows whose keys lay in several parts: a workgroup per row and head.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_tiles_kernel(const PagedArgs a) {
  const PagedView& view = a.view;
  const int row = blockIdx.x, h = blockIdx.y, b = sequence_of(view, row);
  if (b >= view.batch) return;
  const Sequence seq = sequence(a, b);
  if (row < seq.start || (seq.tokens * a.group <= kFewRows && !a.every)) return;
  const Reach reach = seq.reach(a, row - seq.start);
  const int chunk = seq.chunk(a), part0 = reach.begin / chunk, part1 = reach.end > 0 ? (reach.end - 1) / chunk : 0;
  if (part0 == part1) return;
  const int64_t at = ((int64_t)row * a.heads + h) * a.splits + part0;
  join_parts<T, D>(
      a.partial, a.partial + (int64_t)view.tokens * a.heads * a.splits * D, part1 - part0 + 1, [&](int p) { return at + p; },
      static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)h * D);
}

}  // namespace

int launch_tiles(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream) {
  const bool small = a.view.page_shift < 4;
  auto launch = [&](auto kernel, auto join, int rows, int threads) {
    // (at most so many blocks of rows: a part of one per sequence is a block of its own)
    const int64_t blocks = (int64_t)a.view.tokens * a.group / rows + std::min(a.view.batch, a.view.tokens);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks * a.view.kv_heads), 1, (unsigned)a.splits), dim3(threads), 0, stream, a);
    if (a.splits > 1) hipLaunchKernelGGL(join, dim3((unsigned)a.view.tokens, (unsigned)a.heads), dim3(256), 0, stream, a);
  };
  TTMI_DISPATCH_FLOAT(dtype, T, {
    auto sized = [&](auto d) {
      constexpr int D = decltype(d)::value;
      if constexpr (sizeof(T) == 2) {
        if (small) launch(steps_kernel<T, D, true>, join_tiles_kernel<T, D>, kStepRows, 512);
        else launch(steps_kernel<T, D, false>, join_tiles_kernel<T, D>, kStepRows, 512);
      } else {
        if (small) launch(tiles_kernel<T, D, true>, join_tiles_kernel<T, D>, kTileRows, 256);
        else launch(tiles_kernel<T, D, false>, join_tiles_kernel<T, D>, kTileRows, 256);
      }
    };
    if (head_dim == 64) sized(std::integral_constant<int, 64>{});
    else sized(std::integral_constant<int, 128>{});
  });
  return launch_status("paged_attention");
}

}  // namespace ttmi
