// The kernels of paged_tiles.h for rows that see a window or all keys, and sequences on their own; what joins their parts.
#include "paged_tiles.h"

namespace ttmi {
namespace {

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
