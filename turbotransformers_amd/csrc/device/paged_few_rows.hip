// Attention over pages where a sequence has few rows (new tokens times query heads of a key/value head): decoding.
//
// What it has to read, every key and value once, bounds it.  A workgroup has up to 16 rows of one sequence and head and a part of the keys; its four wavefronts
// take every fourth tile of it, each with a running maximum, sum and output of its own, without a barrier until they meet at the end.  Scores are computed transposed,
//     St[key, row] = K[key, :] . Q[row, :]        v_mfma_f32_16x16x32 (fp32: 16x16x4), K as it comes from memory, a 16-byte piece of a row a lane,
// so a lane has one row and four keys of each 16: the statistics need one exchange over the four quarters of the wavefront, and the probabilities lie as the
// second operand of
//     Ot[d, row] += Vt[d, keys] . Pt[keys, row]
// wants them: its order of keys is ours to choose.  Vt is what the transposing reads give of a tile that lies in LDS row by row as it came (fp32: plain reads of a
// column).  Tiles are fetched into registers one ahead: 8 KB of keys and as many of values per wavefront are on their way while one is worked on.
#include "paged_attention.h"

namespace ttmi {
namespace {

template <typename T, int D>
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
  static constexpr int kMergeBytes = 4 * kFewRows * kPitch * 4;
  static constexpr int kLds = 4 * kValueBytes > kMergeBytes ? 4 * kValueBytes : kMergeBytes;
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

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void few_rows_kernel(const PagedArgs a) {
  using S = FewRows<T, D>;
  __shared__ __align__(16) char smem[S::kLds];
  __shared__ float met[4][kFewRows][2];  // maximum and sum of each wavefront's rows
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, b = blockIdx.x / view.kv_heads, part = blockIdx.z;
  const Sequence seq = sequence(a, b);
  const int rows_all = seq.tokens * a.group;
  if (rows_all <= 0 || (rows_all > kFewRows && !a.every)) return;
  const bool whole = rows_all > kFewRows;  // (of these sequences the first part's workgroup takes everything)
  if (whole && part != 0) return;
  const int chunk = whole ? INT32_MAX : seq.chunk(a);
  if (part == 0 && kv_head == 0 && threadIdx.x == 0 && view.lengths[b] > seq.length) page_error(view);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 15, quarter = lane >> 4;
  const T* const q = static_cast<const T*>(a.q);
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  PageCursor cursor;
  cursor.table = view.table + (int64_t)b * view.table_pitch;
  cursor.entry = 0;
  char* const tile = smem + wave * S::kValueBytes;

  for (int row0 = 0; row0 < rows_all; row0 += kFewRows) {
    const int rows = min(kFewRows, rows_all - row0);
    const int token0 = row0 / a.group, token1 = (row0 + rows - 1) / a.group;
    const int token = row < rows ? (row0 + row) / a.group : token0, head = kv_head * a.group + (row < rows ? row0 + row - token * a.group : 0);
    const Reach mine = seq.reach(a, token), low = seq.reach(a, token0), high = seq.reach(a, token1);
    // Keys that some row sees, and those that all rows see: both ends rise with the position.  (A row without keys, before the first one, begins and ends at 0.)
    const int first = low.begin, end = max(low.end, high.end), sure_first = high.begin, sure_end = low.end;
    const int lo = max(part * (int64_t)chunk, (int64_t)(first & ~(S::kKeys - 1))), hi = (int)min((part + 1) * (int64_t)chunk, (int64_t)end);
    if (lo >= hi && part != 0) return;
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
    const bool small_pages = view.page_shift < 4;
    auto load_keys = [&](int key) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) {
        const T* p;
        if (!small_pages) p = keys + group_offset<D>(view, cursor, kv_head, key + 16 * g) + row * D;
        else p = keys + row_offset<D>(view, cursor, kv_head, key + 16 * g + row);
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) kf[g][i] = *reinterpret_cast<const u32x4*>(p + (quarter + 4 * i) * S::kElems);
      }
    };
    auto load_values = [&](int key) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) {
        if (!small_pages) {
          const T* p = values + group_offset<D>(view, cursor, kv_head, key + 16 * g) + lane * S::kElems;
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

    int key = lo + wave * S::kKeys;
    if (key < hi) {
      fetch_pages(view, cursor, min(key >> view.page_shift, cursor.last));
      load_keys(key);
      load_values(key);
    }
    for (; key < hi; key += 4 * S::kKeys) {
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
      const int next = key + 4 * S::kKeys;
      if (next < hi) load_values(next);

      floatx4 st[S::kGroups];
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) {
        st[g] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) st[g] = mma16<T>(kf[g][i], qf[i], st[g]);
      }
      if (next < hi) load_keys(next);
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
      const float moved = fmaxf(top, quarters_max(m) * a.scale_log2e);
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
      if (wild) {  // an infinity or a NaN is what a sum with it is, whatever its weight
#pragma unroll 1
        for (int k = key; k < min(key + S::kKeys, hi); ++k) {
          const T* v = values + row_offset<D>(view, cursor, kv_head, k) + 4 * quarter;
          const bool seen = k >= mine.begin && k < mine.end;
#pragma unroll
          for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = to_float(v[16 * t + e]);
              if (seen && !(fabsf(x) < INFINITY)) ot[t][e] += x;
            }
        }
      }
    }

    // the four wavefronts meet
    sum = quarters_sum(sum);
    __syncthreads();
    float* const stage = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t)
      *reinterpret_cast<floatx4*>(stage + (wave * kFewRows + row) * S::kPitch + 16 * t + 4 * quarter) = ot[t];
    if (quarter == 0) met[wave][row][0] = top, met[wave][row][1] = sum;
    __syncthreads();
    {
      constexpr int kWide = D / 16;  // columns of a thread
      const int r = tid >> 4, d0 = (tid & 15) * kWide;
      if (r < rows) {
        float best = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) best = fmaxf(best, met[w][r][0]);
        const float zero = best == -INFINITY ? 0.f : best;
        float total = 0.f, o[kWide] = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float weight = __builtin_amdgcn_exp2f(met[w][r][0] - zero);
          total += met[w][r][1] * weight;
#pragma unroll
          for (int c = 0; c < kWide; ++c) o[c] += stage[(w * kFewRows + r) * S::kPitch + d0 + c] * weight;
        }
        const int t = (row0 + r) / a.group, h = kv_head * a.group + row0 + r - t * a.group;
        const Reach reach = seq.reach(a, t);
        const int part0 = reach.begin / chunk, part1 = reach.end > 0 ? (reach.end - 1) / chunk : 0;
        if (part0 == part1) {
          if (part == part0) {
            const float inv = total != 0.f ? 1.0f / total : 0.f;
            T* to = static_cast<T*>(a.out) + (seq.start + t) * a.out_pitch + (int64_t)h * D + d0;
            Vec<T, kWide> x;
#pragma unroll
            for (int c = 0; c < kWide; ++c) x.v[c] = from_float<T>(o[c] * inv);
            store_vec<T, kWide>(to, x);
          }
        } else {
          const int64_t at = (((int64_t)b * view.kv_heads + kv_head) * kFewRows + r) * a.splits + part;
#pragma unroll
          for (int c = 0; c < kWide; ++c) a.partial[at * D + d0 + c] = o[c];
          if (d0 == 0) {
            float* ml = a.partial + a.partial_rows * a.splits * D + at * 2;
            ml[0] = best, ml[1] = total;
          }
        }
      }
    }
    if (row0 + kFewRows < rows_all) __syncthreads();
  }
}

// Rows whose keys lay in several parts: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_few_rows_kernel(const PagedArgs a) {
  constexpr int kWide = D / 16;
  const PagedView& view = a.view;
  const int kv_head = blockIdx.x % view.kv_heads, b = blockIdx.x / view.kv_heads;
  const Sequence seq = sequence(a, b);
  const int rows = seq.tokens * a.group, r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * kWide;
  if (rows > kFewRows || r >= rows) return;
  const int t = r / a.group, h = kv_head * a.group + r - t * a.group;
  const Reach reach = seq.reach(a, t);
  const int chunk = seq.chunk(a), part0 = reach.begin / chunk, part1 = reach.end > 0 ? (reach.end - 1) / chunk : 0;
  if (part0 == part1) return;
  const int64_t at = (((int64_t)b * view.kv_heads + kv_head) * kFewRows + r) * a.splits;
  const float* o = a.partial + at * D + d0;
  const float* ml = a.partial + a.partial_rows * a.splits * D + at * 2;
  float best = -INFINITY;
  for (int p = part0; p <= part1; ++p) best = fmaxf(best, ml[2 * p]);
  const float zero = best == -INFINITY ? 0.f : best;
  float total = 0.f, sum[kWide] = {};
#pragma unroll 4
  for (int p = part0; p <= part1; ++p) {
    const float weight = __builtin_amdgcn_exp2f(ml[2 * p] - zero);
    total += ml[2 * p + 1] * weight;
    const Vec<float, kWide> x = load_vec<float, kWide>(o + (int64_t)p * D);
#pragma unroll
    for (int c = 0; c < kWide; ++c) sum[c] += x.v[c] * weight;
  }
  const float inv = total != 0.f ? 1.0f / total : 0.f;
  Vec<T, kWide> x;
#pragma unroll
  for (int c = 0; c < kWide; ++c) x.v[c] = from_float<T>(sum[c] * inv);
  store_vec<T, kWide>(static_cast<T*>(a.out) + (seq.start + t) * a.out_pitch + (int64_t)h * D + d0, x);
}

}  // namespace

int launch_few_rows(const PagedArgs& a, int dtype, int64_t head_dim, hipStream_t stream) {
  const unsigned pairs = (unsigned)((int64_t)a.view.batch * a.view.kv_heads);
  TTMI_DISPATCH_FLOAT(dtype, T, {
    auto launch = [&](auto kernel, auto join) {
      hipLaunchKernelGGL(kernel, dim3(pairs, 1, (unsigned)a.splits), dim3(256), 0, stream, a);
      if (a.splits > 1) hipLaunchKernelGGL(join, dim3(pairs), dim3(256), 0, stream, a);
    };
    if (head_dim == 64) launch(few_rows_kernel<T, 64>, join_few_rows_kernel<T, 64>);
    else launch(few_rows_kernel<T, 128>, join_few_rows_kernel<T, 128>);
  });
  return launch_status("paged_attention");
}

}  // namespace ttmi
