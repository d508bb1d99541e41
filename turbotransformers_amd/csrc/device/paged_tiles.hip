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
__device__ __forceinline__ int value_piece(int row, int piece) {
  if constexpr (sizeof(T) == 4) return piece ^ (((row >> 2) & 1) << 3);
  else if constexpr (D == 128) return piece ^ ((row & 3) << 2);
  else return piece ^ (((row >> 1) & 1) << 2);
}

// A row's sums over one part of its keys: divided and stored, or, where its keys lie in several parts, kept for the kernel that joins those.
template <typename T, int D>
__device__ __forceinline__ void store_rows(const PagedArgs& a, const Sequence& seq, int token, int head, int part, int part0, int part1, bool sees, int lhalf,
                                           const floatx16 (&ot)[D / 32], float top, float sum) {
  const int64_t at_token = seq.start + token;
  if (part0 == part1) {
    if (part != part0) return;
    const float inv = inverse_sum(sum, sees);
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
  const int64_t at = (at_token * a.heads + head) * a.splits + part % a.splits;
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

// SMALL: pages of fewer than 16 slots
template <typename T, int D, bool SMALL>
__global__ __launch_bounds__(256, 2) void tiles_kernel(const PagedArgs a) {
  using S = Tiles<T, D>;
  __shared__ __align__(16) char smem[4 * S::kBytes];
  __shared__ int wild;  // whether values that only some rows see hold infinities or NaNs
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads;
  int b, block;
  if (!find_block(a, blockIdx.x / view.kv_heads, &b, &block)) return;
  const Sequence seq = sequence(a, b);
  const int chunk = seq.chunk(a);
  const int row0 = block * kTileRows, rows = min(kTileRows, seq.tokens * a.group - row0);
  if (blockIdx.z == 0 && kv_head == 0 && block == 0 && threadIdx.x == 0 && view.lengths[b] > seq.length) page_error(view);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lrow = lane & 31, lhalf = lane >> 5;
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  // keys that some row of the workgroup sees, and those that all see (both ends rise with the position); the same of this wavefront
  const Reach low = seq.reach(a, row0 / a.group), high = seq.reach(a, (row0 + rows - 1) / a.group);
  const int first = low.begin, end = max(low.end, high.end), sure_first = high.begin, sure_end = low.end;
  const int part0 = first / chunk, part = part0 + (int)blockIdx.z;
  const int lo = (int)max(part * (int64_t)chunk, (int64_t)(first & ~(S::kKeys - 1))), hi = (int)min((part + 1) * (int64_t)chunk, (int64_t)end);
  if (lo >= hi && part != part0) return;
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
  auto key_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * S::kBytes; };
  auto value_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * S::kBytes + S::kBytes; };
  auto store_piece = [&](int i, int s, int set) __attribute__((always_inline)) {
    const int at = i * 4096 + tid * 16, r = at / S::kRowBytes, c = at % S::kRowBytes / 16;
    *reinterpret_cast<u32x4*>(key_stage(s) + r * S::kRowBytes + key_piece<T, D>(r, c) * 16) = kr[set][i];
    *reinterpret_cast<u32x4*>(value_stage(s) + r * S::kRowBytes + value_piece<T, D>(r, c) * 16) = vr[set][i];
  };
  // Keys that no row sees may hold anything: their values count as zeros.  Where only some rows see a key, infinities and NaNs of its values must not
  // reach the others: they are left out here, noted, and added where they are seen.
  auto partly_seen = [&](int key) __attribute__((always_inline)) { return key < sure_first || key + S::kKeys > sure_end; };
  auto clean_values = [&](int key, int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int k = key + (i * 4096 + tid * 16) / S::kRowBytes;
      if (k < first || k >= end) vr[set][i] = u32x4{0u, 0u, 0u, 0u};
      if (not_finite<T>(vr[set][i])) wild = 1;
      vr[set][i] = finite_part<T>(vr[set][i]);
    }
  };
  if (lo < hi) {
    // (Loads past the last tile fetch that once more, out of L2: a load that may or may not have been sent would make the compiler wait for all of them.)
    const int last = lo + (hi - 1 - lo) / S::kKeys * S::kKeys;
    if constexpr (!SMALL) fetch_pages<S::kRowBytes>(view, cursor, kv_head, lo);
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) load_piece(i, lo, 0);
    if (tid == 0) wild = 0;
    __syncthreads();
    if (partly_seen(lo)) clean_values(lo, 0);
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) store_piece(i, 0, 0);
#pragma unroll
    for (int n = 1; n <= S::kDepth; ++n)
#pragma unroll
      for (int i = 0; i < S::kPieces; ++i) load_piece(i, min(lo + n * S::kKeys, last), n % S::kDepth);  // (in the same 64 pages)
    __syncthreads();
    // One tile; its stage is known to the compiler, so that places in LDS are fixed numbers behind one of the lane's.
    auto work_on = [&](int key, auto stage) __attribute__((always_inline)) {
      constexpr int s = decltype(stage)::value;
      // The other stage is free: what was fetched for it while the last tile was worked on goes there, and the tile behind it is sent for.
      constexpr int set = (s + 1) % S::kDepth;
      const int after = min(key + (1 + S::kDepth) * S::kKeys, last);
      if constexpr (!SMALL) come_to<S::kRowBytes>(view, cursor, kv_head, after);
      if (__builtin_expect(partly_seen(key + S::kKeys), 0)) clean_values(key + S::kKeys, set);
      if (key >= wave_end || key + S::kKeys <= wave_first) {  // nothing to do for this wavefront's rows
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
        if (n < S::kPieces) store_piece(n, s ^ 1, set);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < S::kPieces; ++i) load_piece(i, after, set);
      if (__builtin_expect(key < wave_high.begin || key + S::kKeys > wave_low.end, 0)) {
        const int from = mine.begin - key - 4 * lhalf;
        const uint32_t span = (uint32_t)(mine.end - mine.begin);
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((uint32_t)(32 * u + 8 * (e / 4) + e % 4 - from) >= span) st[u][e] = -INFINITY;
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
        static_assert(sizeof(T) == 2 || S::kSubs == 1, "32 keys");
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          st[0][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[0][e], a.scale_log2e, -zero));
          sum += st[0][e];
        }
        auto read_value = [&](int n) __attribute__((always_inline)) {  // the operand of the n-th matrix instruction of Ot: kOut of them for each pair of keys
          const int e = n / S::kOut, r = 8 * (e / 4) + 4 * lhalf + e % 4;
          return *reinterpret_cast<const float*>(vt + r * S::kRowBytes + value_piece<T, D>(r, 8 * (n % S::kOut) + (lrow >> 2)) * 16 + (lrow & 3) * 4);
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
        for (int k = key; k < min(key + S::kKeys, hi); ++k) {
          const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * lhalf;
          const bool seen = k >= mine.begin && k < mine.end;
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
  const bool sees = mine.end > 0;
  store_rows<T, D>(a, seq, token, head, part, sees ? mine.begin / chunk : part0, sees ? (mine.end - 1) / chunk : part0, sees, lhalf, ot, top, sum);
}

// Rows whose keys lay in several parts.  What their bytes take is little; what counts is how many trips to memory follow one another: the sequence, its length, the parts.  So
// a thread has four columns of a row and head and asks for up to MOST parts at once.  (us for two parts, 32 heads of 64: a wavefront per row and head 10.4 for 600 tokens and 14.8
// for 1000, this 4.9 for 700.)  MOST 0, many parts: a workgroup per row and head, whose threads share them.
constexpr int kFewParts = 16;
template <typename T, int D, int MOST>
__global__ __launch_bounds__(256) void join_tiles_kernel(const PagedArgs a) {
  const PagedView& view = a.view;
  const int row = blockIdx.x, b = sequence_of(view, row);
  if (b >= view.batch) return;
  const Sequence seq = sequence(a, b);
  if (row < seq.start || (seq.tokens * a.group <= kFewRows && !a.every)) return;
  const Reach reach = seq.reach(a, row - seq.start);
  const int chunk = seq.chunk(a), part0 = reach.begin / chunk, parts = (reach.end > 0 ? (reach.end - 1) / chunk : 0) - part0 + 1;
  if (parts <= 1) return;
  const float* const met = a.partial + (int64_t)view.tokens * a.heads * a.splits * D;
  if constexpr (MOST == 0) {
    const int h = blockIdx.y;
    const int64_t at = ((int64_t)row * a.heads + h) * a.splits;
    join_parts<T, D>(
        a.partial, met, parts, true, [&](int p) { return at + (part0 + p) % a.splits; }, static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)h * D);
  } else {
    constexpr int kThreads = D / 4;
    const int h = blockIdx.y * (256 / kThreads) + threadIdx.x / kThreads, d0 = threadIdx.x % kThreads * 4;
    if (h >= a.heads) return;
    const int64_t at = ((int64_t)row * a.heads + h) * a.splits;
    floatx4 x[MOST];
    floatx2 ml[MOST];
#pragma unroll
    for (int p = 0; p < MOST; ++p)
      if (p < parts) {
        const int64_t from = at + (part0 + p) % a.splits;
        x[p] = *reinterpret_cast<const floatx4*>(a.partial + from * D + d0);
        ml[p] = *reinterpret_cast<const floatx2*>(met + from * 2);
      }
    float best = -INFINITY, total = 0.f;
#pragma unroll
    for (int p = 0; p < MOST; ++p)
      if (p < parts) best = fmaxf(best, ml[p][0]);
    const float zero = best == -INFINITY ? 0.f : best;
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < MOST; ++p)
      if (p < parts) {
        const float weight = __builtin_amdgcn_exp2f(ml[p][0] - zero);
        total += ml[p][1] * weight;
        sum += x[p] * weight;
      }
    const float inv = inverse_sum(total, true);  // (a row of several parts sees keys)
    Vec<T, 4> y;
#pragma unroll
    for (int c = 0; c < 4; ++c) y.v[c] = from_float<T>(sum[c] * inv);
    store_vec<T, 4>(static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)h * D + d0, y);
  }
}

}  // namespace

int launch_tiles(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream) {
  // (at most so many blocks of rows: a part of one per sequence is a block of its own)
  const int64_t blocks = (int64_t)a.view.tokens * a.group / kTileRows + std::min(a.view.batch, a.view.tokens);
  const bool small = a.view.page_shift < 4;
  PagedArgs args = a;
  args.ordered = blocks * a.view.kv_heads * a.splits > 2 * compute_units();
  TTMI_DISPATCH_FLOAT(dtype, T, {
    auto launch = [&](auto d, auto small_pages) {
      constexpr int D = decltype(d)::value;
      hipLaunchKernelGGL((tiles_kernel<T, D, decltype(small_pages)::value>), dim3((unsigned)(blocks * a.view.kv_heads), 1, (unsigned)a.splits), dim3(256), 0, stream, args);
      const unsigned tokens = (unsigned)a.view.tokens, few = (unsigned)ceil_div(a.heads, 256 / (D / 4));
      if (a.splits > kFewParts) hipLaunchKernelGGL((join_tiles_kernel<T, D, 0>), dim3(tokens, a.heads), dim3(256), 0, stream, a);
      else if (a.splits > 2) hipLaunchKernelGGL((join_tiles_kernel<T, D, kFewParts>), dim3(tokens, few), dim3(256), 0, stream, a);
      else if (a.splits > 1) hipLaunchKernelGGL((join_tiles_kernel<T, D, 2>), dim3(tokens, few), dim3(256), 0, stream, a);
    };
    const std::integral_constant<int, 64> d64;
    const std::integral_constant<int, 128> d128;
    if (head_dim == 64 && small) launch(d64, std::true_type{});
    else if (head_dim == 64) launch(d64, std::false_type{});
    else if (small) launch(d128, std::true_type{});
    else launch(d128, std::false_type{});
  });
  return launch_status("paged_attention");
}

}  // namespace ttmi
