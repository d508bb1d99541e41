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

// The `want`-th block of rows of all sequences -> its sequence and number in it (false: there are fewer).  Every lane looks at a sequence.
__device__ __forceinline__ bool find_block(const PagedArgs& a, int want, int* b, int* block) {
  const int lane = (int)(threadIdx.x % kWave);
  for (int base = 0; base < a.view.batch; base += kWave) {
    int blocks = 0;
    if (base + lane < a.view.batch) {
      const int rows = sequence(a, base + lane).tokens * a.group;
      if (rows > kFewRows || a.every) blocks = (rows + kTileRows - 1) / kTileRows;
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

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void tiles_kernel(const PagedArgs a) {
  using S = Tiles<T, D>;
  __shared__ __align__(16) char smem[4 * S::kBytes];
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, part = blockIdx.z;
  int b, block;
  if (!find_block(a, blockIdx.x / view.kv_heads, &b, &block)) return;
  const Sequence seq = sequence(a, b);
  const int chunk = seq.chunk(a);
  const int row0 = block * kTileRows, rows = min(kTileRows, seq.tokens * a.group - row0);
  if (part == 0 && kv_head == 0 && block == 0 && threadIdx.x == 0 && view.lengths[b] > seq.length) page_error(view);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lrow = lane & 31, lhalf = lane >> 5;
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
  cursor.first = 0, cursor.entry = 0, cursor.ahead = 0;
  const bool small_pages = view.page_shift < 4;
  u32x4 kr[S::kPieces], vr[S::kPieces];
  // 16-byte pieces of a tile: thread by thread, 4 KB after 4 KB.  A wavefront's 1 KB lies in one group of 16 rows.
  auto load_tile = [&](int key) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int at = i * 4096 + tid * 16, r = at / S::kRowBytes, c = at % S::kRowBytes / (int)sizeof(T);
      int64_t from;
      if (!small_pages) {
        const int group = __builtin_amdgcn_readfirstlane(i * 4096 + wave * 1024) / S::kRowBytes & ~15;
        from = group_offset<D>(view, cursor, kv_head, key + group) + (r - group) * D + c;
      } else {
        from = row_offset<D>(view, cursor, kv_head, key + r) + c;
      }
      kr[i] = *reinterpret_cast<const u32x4*>(keys + from);
      vr[i] = *reinterpret_cast<const u32x4*>(values + from);
    }
  };
  auto key_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * S::kBytes; };
  auto value_stage = [&](int s) __attribute__((always_inline)) { return smem + s * 2 * S::kBytes + S::kBytes; };
  // Keys that no row sees may hold anything: their values count as zeros.  Where only some rows see a key, infinities and NaNs of its values must not
  // reach the others: they are left out here (-> whether there are any) and added where they are seen.
  auto store_tile = [&](int key, int s) __attribute__((always_inline)) {
    uint32_t wild = 0;
    if (key < sure_first || key + S::kKeys > sure_end) {
#pragma unroll
      for (int i = 0; i < S::kPieces; ++i) {
        const int k = key + (i * 4096 + tid * 16) / S::kRowBytes;
        if (k < first || k >= end) vr[i] = u32x4{0u, 0u, 0u, 0u};
        wild |= not_finite<T>(vr[i]);
        vr[i] = finite_part<T>(vr[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < S::kPieces; ++i) {
      const int at = i * 4096 + tid * 16, r = at / S::kRowBytes, c = at % S::kRowBytes / 16;
      *reinterpret_cast<u32x4*>(key_stage(s) + r * S::kRowBytes + key_piece<T, D>(r, c) * 16) = kr[i];
      *reinterpret_cast<u32x4*>(value_stage(s) + r * S::kRowBytes + value_piece<T, D>(r, c) * 16) = vr[i];
    }
    return wild;
  };
  auto barrier = [&](int key, uint32_t wild) __attribute__((always_inline)) -> bool {
    if (key < sure_first || key + S::kKeys > sure_end) return __syncthreads_or((int)wild) != 0;
    __syncthreads();
    return false;
  };

  bool wild = false;
  int s = 0;
  if (lo < hi) {
    fetch_pages(view, cursor, min(lo >> view.page_shift, cursor.last));
    load_tile(lo);
    const uint32_t w = store_tile(lo, 0);
    if (lo + S::kKeys < hi) load_tile(lo + S::kKeys);
    wild = barrier(lo, w);
  }
  for (int key = lo; key < hi; key += S::kKeys, s ^= 1) {
    if (key < wave_end && key + S::kKeys > wave_first) {
      const char* const kt = key_stage(s);
      const char* const vt = value_stage(s);
      floatx16 st[S::kSubs];
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) st[u][e] = 0.f;
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
          const int r = 32 * u + lrow;
          st[u] = mma32<T>(*reinterpret_cast<const u32x4*>(kt + r * S::kRowBytes + key_piece<T, D>(r, 2 * i + lhalf) * 16), qf[i], st[u]);
        }
      }
      if (key < wave_high.begin || key + S::kKeys > wave_low.end) {
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int k = key + 32 * u + 8 * (e / 4) + 4 * lhalf + e % 4;
            if (k < mine.begin || k >= mine.end) st[u][e] = -INFINITY;
          }
      }
      float m = st[0][0];
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, st[u][e]);
      {
        const LanePair sw = swap_halves(m);
        m = fmaxf(sw.a, sw.b);
      }
      const float moved = fmaxf(top, m * a.scale_log2e);
      const float zero = moved == -INFINITY ? 0.f : moved;  // (a row that has seen no key yet)
      const float shrink = __builtin_amdgcn_exp2f(top - zero);
      top = moved;
      if (__any(shrink != 1.f)) {
        sum *= shrink;
#pragma unroll
        for (int t = 0; t < S::kOut; ++t) ot[t] *= shrink;
      }
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) st[u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[u][e], a.scale_log2e, -zero));
        if constexpr (sizeof(T) == 2) {
          // rounded to the type for the second product; the sum is that of the rounded ones, so what rounding does to all of them alike cancels
          u32x4 pf[2];
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            pf[w >> 2][w & 3] = pack2<T>(st[u][2 * w], st[u][2 * w + 1]);
            sum = add_pair<T>(pf[w >> 2][w & 3], sum);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < S::kOut; ++t) {
              u32x4 v;
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const int r = 32 * u + 16 * i + 8 * g + 4 * lhalf + ((lane >> 2) & 3);
                const u32x2 half =
                    read_transposed(vt + r * S::kRowBytes + value_piece<T, D>(r, 4 * t + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 + (lane & 1) * 8);
                v[2 * g] = half[0], v[2 * g + 1] = half[1];
              }
              ot[t] = mma32<T>(v, pf[i], ot[t]);
            }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sum += st[u][e];
            const int r = 32 * u + 8 * (e / 4) + 4 * lhalf + e % 4;
#pragma unroll
            for (int t = 0; t < S::kOut; ++t) {
              const float v = *reinterpret_cast<const float*>(vt + r * S::kRowBytes + value_piece<T, D>(r, 8 * t + (lrow >> 2)) * 16 + (lrow & 3) * 4);
              ot[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, st[u][e], ot[t], 0, 0, 0);
            }
          }
        }
      }
      if (wild) {  // an infinity or a NaN is what a sum with it is, whatever its weight
#pragma unroll 1
        for (int k = key; k < min(key + S::kKeys, hi); ++k) {
          const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * lhalf;
          const bool seen = k >= mine.begin && k < mine.end;
#pragma unroll
          for (int t = 0; t < S::kOut; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x = to_float(v[32 * t + 8 * (e / 4) + e % 4]);
              if (seen && !(fabsf(x) < INFINITY)) ot[t][e] += x;
            }
        }
      }
    }
    if (key + S::kKeys < hi) {
      const uint32_t w = store_tile(key + S::kKeys, s ^ 1);
      if (key + 2 * S::kKeys < hi) load_tile(key + 2 * S::kKeys);
      wild = barrier(key + S::kKeys, w);
    }
  }

  {
    const LanePair both = swap_halves(sum);
    sum = both.a + both.b;
  }
  if (!live) return;
  const int part0 = mine.begin / chunk, part1 = mine.end > 0 ? (mine.end - 1) / chunk : 0;
  const int64_t at_token = seq.start + token;
  if (part0 == part1) {
    if (part != part0) return;
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    T* to = static_cast<T*>(a.out) + at_token * a.out_pitch + (int64_t)head * D + 4 * lhalf;
#pragma unroll
    for (int t = 0; t < S::kOut; ++t)
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
  for (int t = 0; t < S::kOut; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<floatx4*>(to + 32 * t + 8 * g) = floatx4{ot[t][4 * g], ot[t][4 * g + 1], ot[t][4 * g + 2], ot[t][4 * g + 3]};
  if (lhalf == 0) {
    float* ml = a.partial + (int64_t)view.tokens * a.heads * a.splits * D + at * 2;
    ml[0] = top, ml[1] = sum;
  }
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
  // (at most so many blocks of rows: a part of one per sequence is a block of its own)
  const int64_t blocks = (int64_t)a.view.tokens * a.group / kTileRows + std::min(a.view.batch, a.view.tokens);
  TTMI_DISPATCH_FLOAT(dtype, T, {
    auto launch = [&](auto kernel, auto join) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks * a.view.kv_heads), 1, (unsigned)a.splits), dim3(256), 0, stream, a);
      if (a.splits > 1) hipLaunchKernelGGL(join, dim3((unsigned)a.view.tokens, (unsigned)a.heads), dim3(256), 0, stream, a);
    };
    if (head_dim == 64) launch(tiles_kernel<T, 64>, join_tiles_kernel<T, 64>);
    else launch(tiles_kernel<T, 128>, join_tiles_kernel<T, 128>);
  });
  return launch_status("paged_attention");
}

}  // namespace ttmi
