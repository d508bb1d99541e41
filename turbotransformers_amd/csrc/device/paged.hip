// A decoder's keys and values in pages: new tokens turned by their positions and stored, pages copied.
#include "paged.h"

#include <new>
#include <utility>
#include <vector>

namespace ttmi {

// ---- rotary positions and the append to the cache ---------------------------------------------------------------------
// theta = position * inv_freq;  y1 = x1 cos theta - x2 sin theta, y2 = x1 sin theta + x2 cos theta.
// The angle is formed in 64 bits and taken to a fraction of a turn there, since at position 10^6 a 32-bit angle is off by up to 2^-5; what is left, at most an
// eighth of a turn from the nearest quarter, goes through the Taylor sums of sine and cosine (|x| <= pi/4: the first terms left out are
// x^11/11! < 2e-9 and x^12/12! < 2e-10).  All heads of a token turn by the same angles, so a workgroup computes them once, into LDS.
// Bytes bound it: each row is read and written once, 16 bytes a lane.  6 chunks of 512 to 4096 tokens, 32 + 8 + 8 heads of 128, bf16: 45.7 us from HBM (4.2 TB/s), 33 from the
// last-level cache; a token of each of 8 sequences 3.5, trips to memory that follow one another (sequence, position, page).
__device__ __forceinline__ float2 unit_turn(double angle) {
  const double turns = angle * 0.15915494309189533577;  // 1 / 2 pi
  const double part = turns - rint(turns);
  const double quarter = rint(part * 4.0);
  const float x = (float)((part - quarter * 0.25) * 6.283185307179586477);
  const float z = x * x;
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(z, s, 8.3333333e-3f);
  s = __builtin_fmaf(z, s, -1.6666667e-1f);
  s = __builtin_fmaf(z * s, x, x);
  float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(z, c, -1.3888889e-3f);
  c = __builtin_fmaf(z, c, 4.1666667e-2f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const int q = (int)quarter & 3;  // -2 .. 2 quarters
  const float a = (q & 1) ? s : c, b = (q & 1) ? c : s;
  return make_float2((q == 1 || q == 2) ? -a : a, (q & 2) ? -b : b);
}

// One workgroup: the items first, first + step, ... of one token.  An item is W elements of a head, or the two halves' W elements of
// W pairs; a head of queries or keys has `items` of them.
template <typename T, int W, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_append_kernel(const T* qkv, int64_t qkv_pitch, T* q_out, int64_t q_pitch, int heads,
                                                            T* __restrict__ keys, T* __restrict__ values, const PagedView view,
                                                            const double* __restrict__ inv_freq, int half, float amplitude) {
  const int token = blockIdx.x;
  const int b = sequence_of(view, token);
  if (b >= view.batch) return;
  const int start = view.starts[b];
  if (token < start) return;
  const int position = view.lengths[b] - view.starts[b + 1] + token;
  __shared__ float2 turn[128];
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    const float2 u = unit_turn((double)position * inv_freq[i]);
    turn[i] = make_float2(u.x * amplitude, u.y * amplitude);
  }
  __syncthreads();

  const int d = view.head_dim, hk = view.kv_heads;
  bool stored = position >= 0 && (position >> view.page_shift) < view.table_pitch;
  int page = 0;
  if (stored) {
    page = view.table[(int64_t)b * view.table_pitch + (position >> view.page_shift)];
    stored = (unsigned)page < (unsigned)view.pages;
  }
  if (!stored && threadIdx.x == 0) page_error(view);
  const int slot = position & ((1 << view.page_shift) - 1);
  // row of head 0; the heads of a page lie page_size rows apart
  const int64_t row0 = (((int64_t)page * hk) << view.page_shift) + slot;

  const int pairs = INTERLEAVED ? 0 : half / W;     // items of a head that are two halves
  const int items = d / W - pairs, plain = d / W;   // of a head of queries or keys, and of values
  const int turned = (heads + hk) * items, all = turned + hk * plain;
  const T* in = qkv + (int64_t)token * qkv_pitch;
  T* q_row = q_out + (int64_t)token * q_pitch;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < all; i += gridDim.y * blockDim.x) {
    const bool value = i >= turned;
    const int j = value ? i - turned : i, per = value ? plain : items;
    const int head = j / per, item = j - head * per;
    const int from = value ? heads + hk + head : head;
    const T* x = in + (int64_t)from * d;
    T* y;
    if (!value && head < heads) y = q_row + (int64_t)head * d;
    else {
      if (!stored) continue;
      const int kv = value ? head : head - heads;
      y = (value ? values : keys) + (row0 + ((int64_t)kv << view.page_shift)) * d;
    }
    if (!INTERLEAVED && !value && item < pairs) {
      const int at = item * W;
      Vec<T, W> lo = load_vec<T, W>(x + at), hi = load_vec<T, W>(x + half + at);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float2 t = turn[at + e];
        const float x1 = to_float(lo.v[e]), x2 = to_float(hi.v[e]);
        lo.v[e] = from_float<T>(__builtin_fmaf(x1, t.x, -x2 * t.y));
        hi.v[e] = from_float<T>(__builtin_fmaf(x1, t.y, x2 * t.x));
      }
      store_vec<T, W>(y + at, lo);
      store_vec<T, W>(y + half + at, hi);
      continue;
    }
    const int at = (!INTERLEAVED && !value ? item + pairs : item) * W;
    Vec<T, W> x0 = load_vec<T, W>(x + at);
    if (INTERLEAVED && !value && at < 2 * half) {
#pragma unroll
      for (int e = 0; e + 1 < W; e += 2) {
        const float2 t = turn[(at + e) / 2];
        const float x1 = to_float(x0.v[e]), x2 = to_float(x0.v[e + 1]);
        x0.v[e] = from_float<T>(__builtin_fmaf(x1, t.x, -x2 * t.y));
        x0.v[e + 1] = from_float<T>(__builtin_fmaf(x1, t.y, x2 * t.x));
      }
    }
    store_vec<T, W>(y + at, x0);
  }
}

template <typename T, int W, bool INTERLEAVED>
static void launch_rotary_append(const void* qkv, int64_t qkv_pitch, void* q_out, int64_t q_pitch, int heads, const ttmi_paged_cache* cache,
                                 const PagedView& view, const double* inv_freq, int half, float amplitude, hipStream_t stream) {
  const int d = view.head_dim, items = (heads + view.kv_heads) * (d / W - (INTERLEAVED ? 0 : half / W)) + view.kv_heads * (d / W);
  const int parts = (int)std::min<int64_t>(ceil_div(items, 256), 64);
  hipLaunchKernelGGL((rotary_append_kernel<T, W, INTERLEAVED>), dim3(view.tokens, parts), dim3(256), 0, stream, static_cast<const T*>(qkv), qkv_pitch,
                     static_cast<T*>(q_out), q_pitch, heads, static_cast<T*>(cache->keys), static_cast<T*>(cache->values), view, inv_freq, half, amplitude);
}

// ---- pages copied to pages ----------------------------------------------------------------------------------------------
// The list goes along with the launch: nothing is copied to the device, and a recorded call keeps its own.  A page goes through the registers of ceil(bytes / 16 KB) workgroups,
// four pieces of 16 bytes a lane on their way: 901 pages of 64 KB in keys and values of 24 layers 1124 us, 5.05 TB/s (a large copy here 4.8); 4 pages of 24 KB in 12 layers 3.3.
constexpr int kCopyPairs = 448, kCopyFew = 16;  // what fits the arguments of a launch (4 KB); a short list, whose launch is shorter: a call for 1, 4, 16 pairs 5.3 / 4.1, 5.3 / 4.7, 5.5 / 5.1 us
constexpr int kCopyBytes = 16384;  // of a workgroup
template <int N>
struct PagePairs {
  int32_t from[N], to[N];
};

template <int N>
__global__ __launch_bounds__(256) void copy_pages_kernel(char* __restrict__ keys, char* __restrict__ values, int64_t pages, int64_t page_bytes,
                                                         const PagePairs<N> pairs) {
  typedef uint32_t Quad __attribute__((ext_vector_type(4)));
  const int64_t layer = blockIdx.z >> 1;
  char* const base = (blockIdx.z & 1) ? values : keys;
  const int64_t from = (layer * pages + pairs.from[blockIdx.y]) * page_bytes, to = (layer * pages + pairs.to[blockIdx.y]) * page_bytes;
  const int64_t first = (int64_t)blockIdx.x * kCopyBytes + threadIdx.x * 16;
  constexpr int kPieces = kCopyBytes / (256 * 16);
  Quad x[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (first + i * 4096 < page_bytes) x[i] = *reinterpret_cast<const Quad*>(base + from + first + i * 4096);
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (first + i * 4096 < page_bytes) *reinterpret_cast<Quad*>(base + to + first + i * 4096) = x[i];
}

template <int N>
static void launch_copy_pages(void* keys, void* values, int64_t layers, int64_t pages, int64_t page_bytes, const int32_t* sources, const int32_t* destinations,
                              int count, hipStream_t stream) {
  PagePairs<N> pairs;
  std::copy_n(sources, count, pairs.from);
  std::copy_n(destinations, count, pairs.to);
  std::fill(pairs.from + count, pairs.from + N, 0);
  std::fill(pairs.to + count, pairs.to + N, 0);
  const dim3 grid((unsigned)ceil_div(page_bytes, kCopyBytes), count, (unsigned)layers * 2);
  hipLaunchKernelGGL(copy_pages_kernel<N>, grid, dim3(256), 0, stream, static_cast<char*>(keys), static_cast<char*>(values), pages, page_bytes, pairs);
}

}  // namespace ttmi

using namespace ttmi;

extern "C" {

int ttmi_rotary_append(const void* qkv, int64_t qkv_pitch, void* q_out, int64_t q_pitch, int64_t heads, const ttmi_paged_cache* cache,
                       const ttmi_paged_batch* batch, const double* inv_freq, int64_t rotary_dim, int interleaved, float amplitude,
                       int dtype, void* stream) {
  PagedView view;
  if (int rc = paged_view(cache, batch, heads, &view)) return rc;
  const int64_t d = cache->head_dim;
  TTMI_REQUIRE(rotary_dim >= 0 && rotary_dim <= d && rotary_dim % 2 == 0, "rotary_dim must be even and at most head_dim");
  TTMI_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "inv_freq is null");
  TTMI_REQUIRE(qkv_pitch >= (heads + 2 * cache->kv_heads) * d && q_pitch >= heads * d, "rows overlap: a pitch is too small");
  TTMI_REQUIRE(dtype == TTMI_F32 || dtype == TTMI_F16 || dtype == TTMI_BF16, "unsupported dtype");
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  TTMI_REQUIRE(qkv != nullptr && q_out != nullptr, "qkv or q_out is null");
  TTMI_REQUIRE(q_out != qkv || q_pitch == qkv_pitch, "queries turned in place keep their pitch");
  const int half = (int)(rotary_dim / 2), wide = 16 / (int)dtype_size(dtype);
  const bool vectors = rows_aligned(qkv, qkv_pitch, dtype) && rows_aligned(q_out, q_pitch, dtype) &&
                       (interleaved ? rotary_dim : half) % wide == 0;
  // (rows that are not aligned to 16 bytes, and parts of a head that are no whole pieces, go by the element or the pair)
  TTMI_REQUIRE(((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & (dtype_size(dtype) - 1)) == 0, "qkv or q_out is not aligned to its elements");
  const bool pairs_aligned = ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & (2 * dtype_size(dtype) - 1)) == 0 &&
                             qkv_pitch % 2 == 0 && q_pitch % 2 == 0;
  TTMI_REQUIRE(!interleaved || vectors || pairs_aligned, "interleaved pairs must be aligned to two elements");
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define TTMI_APPEND(W, I) launch_rotary_append<T, W, I>(qkv, qkv_pitch, q_out, q_pitch, (int)heads, cache, view, inv_freq, half, amplitude, s)
  TTMI_DISPATCH_FLOAT(dtype, T, {
    constexpr int kWide = 16 / (int)sizeof(T);
    if (vectors && interleaved) TTMI_APPEND(kWide, true);
    else if (vectors) TTMI_APPEND(kWide, false);
    else if (interleaved) TTMI_APPEND(2, true);
    else TTMI_APPEND(1, false);
  });
#undef TTMI_APPEND
  return launch_status("rotary_append");
}

int ttmi_copy_pages(void* keys, void* values, int64_t layers, int64_t pages, int64_t page_bytes, const int32_t* sources,
                    const int32_t* destinations, int64_t count, void* stream) {
  TTMI_REQUIRE(layers >= 0 && layers <= 32767 && pages >= 0 && pages <= INT32_MAX && count >= 0, "bad number of layers, pages or copies");
  TTMI_REQUIRE(page_bytes >= 0 && page_bytes % 16 == 0 && page_bytes <= (1ll << 36), "page_bytes must be a multiple of 16, at most 2^36");
  if (count == 0 || layers == 0 || page_bytes == 0) return 0;
  TTMI_REQUIRE(keys != nullptr && values != nullptr && sources != nullptr && destinations != nullptr, "keys, values, sources or destinations is null");
  TTMI_REQUIRE(((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 15) == 0, "keys and values must be 16-byte aligned");
  try {
    // 1: a source, 2: a destination
    std::vector<std::pair<int32_t, int>> uses;
    uses.reserve(2 * (size_t)count);
    for (int64_t i = 0; i < count; ++i) {
      TTMI_REQUIRE(sources[i] >= 0 && sources[i] < pages && destinations[i] >= 0 && destinations[i] < pages, "a page is outside the cache");
      uses.emplace_back(sources[i], 1);
      uses.emplace_back(destinations[i], 2);
    }
    std::sort(uses.begin(), uses.end());
    for (size_t i = 1; i < uses.size(); ++i)
      TTMI_REQUIRE(uses[i].first != uses[i - 1].first || uses[i].second == 1, "a page is a destination twice, or a source and a destination");
  } catch (const std::bad_alloc&) {
    return fail(TTMI_ENOMEM, "no memory for the list of copies");
  }
  for (int64_t at = 0; at < count; at += kCopyPairs) {
    const int n = (int)std::min<int64_t>(kCopyPairs, count - at);
    const auto launch = count <= kCopyFew ? launch_copy_pages<kCopyFew> : launch_copy_pages<kCopyPairs>;
    launch(keys, values, layers, pages, page_bytes, sources + at, destinations + at, n, static_cast<hipStream_t>(stream));
    if (int rc = launch_status("copy_pages")) return rc;
  }
  return 0;
}

}  // extern "C"
