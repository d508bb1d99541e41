// Attention over pages where tokens see a window and the first keys of their sequence: o = sum_j p_j v_j, p = softmax_j(scale q . k_j) over the keys j that a token sees.
// A wavefront has one token and head and goes over the keys 64 at a time, a lane each: scores, the running maximum and sum, then the lanes take columns of the values.
#include <limits>

#include "paged_attention.h"

namespace ttmi {
namespace {

template <typename T, int D>
__global__ __launch_bounds__(64) void sight_kernel(const PagedArgs a, int sinks) {
  const PagedView& view = a.view;
  const int row = blockIdx.x, head = blockIdx.y, kv_head = head / a.group, lane = threadIdx.x;
  const int b = sequence_of(view, row);
  if (b >= view.batch) return;
  const Sequence seq = sequence(a, b);
  if (row < seq.start) return;
  if (lane == 0 && head == 0 && view.lengths[b] > seq.length) page_error(view);
  const Reach reach = seq.reach(a, row - seq.start);
  const int low = a.window > 0 ? min(sinks, reach.end) : 0;  // keys below are seen
  PageCursor cursor;
  cursor.table = view.table + (int64_t)b * view.table_pitch;
  cursor.last = max(0, (reach.end - 1) >> view.page_shift);
  const T* const keys = static_cast<const T*>(a.keys);
  const T* const values = static_cast<const T*>(a.values);
  __shared__ float q[D], p[64];
  const T* const from = static_cast<const T*>(a.q) + (int64_t)row * a.q_pitch + (int64_t)head * D;
  for (int i = lane; i < D; i += 64) q[i] = to_float(from[i]);
  __syncthreads();
  float top = -INFINITY, sum = 0.f, o[D / 64] = {};
  for (int key = 0; key < reach.end; key += 64) {
    if (key >= low && key + 64 <= reach.begin) continue;
    const int k = key + lane;
    const bool seen = k < reach.end && (k < low || k >= reach.begin);
    float s = -INFINITY;
    if (seen) {
      const T* const x = keys + row_offset<D>(view, cursor, kv_head, k);
      s = 0.f;
      for (int i = 0; i < D; ++i) s = __builtin_fmaf(q[i], to_float(x[i]), s);
      s *= a.scale_log2e;
    }
    float m = s;
    for (int step = 32; step > 0; step /= 2) m = fmaxf(m, __shfl_xor(m, step, kWave));
    m = fmaxf(m, top);
    const float zero = m == -INFINITY ? 0.f : m, shrink = __builtin_amdgcn_exp2f(top - zero);
    top = m;
    const float mine = seen ? __builtin_amdgcn_exp2f(s - zero) : 0.f;
    float all = mine;
    for (int step = 32; step > 0; step /= 2) all += __shfl_xor(all, step, kWave);
    sum = sum * shrink + all;
    p[lane] = mine;
    __syncthreads();
    for (int c = 0; c < D / 64; ++c) o[c] *= shrink;
    for (int j = 0; j < 64 && key + j < reach.end; ++j) {
      if (key + j >= low && key + j < reach.begin) continue;
      const T* const v = values + row_offset<D>(view, cursor, kv_head, key + j);
      for (int c = 0; c < D / 64; ++c) o[c] = __builtin_fmaf(p[j], to_float(v[lane + 64 * c]), o[c]);
    }
    __syncthreads();
  }
  const float inv = inverse_sum(sum, reach.end > 0);
  T* const to = static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)head * D;
  for (int c = 0; c < D / 64; ++c) to[lane + 64 * c] = from_float<T>(o[c] * inv);
}

}  // namespace
}  // namespace ttmi

using namespace ttmi;

extern "C" {

int ttmi_paged_attention_sight_workspace(const ttmi_paged_cache* cache, const ttmi_paged_batch* batch, int64_t heads, int64_t max_tokens, int64_t max_length,
                                         const ttmi_paged_sight* sight, int dtype, int64_t* bytes) {
  TTMI_REQUIRE(sight != nullptr, "sight is null");
  TTMI_REQUIRE(sight->sinks >= 0 && sight->family_count >= 0 && sight->max_shared >= 0, "sinks, family_count and max_shared must not be negative");
  if (sight->families == nullptr && (sight->sinks == 0 || sight->window == 0))
    return ttmi_paged_attention_workspace(cache, batch, heads, max_tokens, max_length, sight->window, dtype, bytes);
  PagedView view;
  TTMI_REQUIRE(bytes != nullptr, "bytes is null");
  if (int rc = paged_view(cache, batch, heads, &view)) return rc;
  TTMI_REQUIRE(sight->window >= 0 && max_tokens >= 0 && max_length >= 0, "window, max_tokens and max_length must not be negative");
  *bytes = 0;
  return 0;
}

int ttmi_paged_attention_sight(const void* q, int64_t q_pitch, void* out, int64_t out_pitch, int64_t heads, const ttmi_paged_cache* cache,
                               const ttmi_paged_batch* batch, int64_t max_tokens, int64_t max_length, float scale, int causal, const ttmi_paged_sight* sight,
                               void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  TTMI_REQUIRE(sight != nullptr, "sight is null");
  TTMI_REQUIRE(sight->sinks >= 0 && sight->family_count >= 0 && sight->max_shared >= 0, "sinks, family_count and max_shared must not be negative");
  if (sight->families == nullptr && (sight->sinks == 0 || sight->window == 0))
    return ttmi_paged_attention(q, q_pitch, out, out_pitch, heads, cache, batch, max_tokens, max_length, scale, causal, sight->window, workspace, workspace_bytes,
                                dtype, stream);
  PagedArgs a;
  if (int rc = paged_view(cache, batch, heads, &a.view)) return rc;
  const int64_t d = cache->head_dim;
  TTMI_REQUIRE(d == 64 || d == 128, "paged attention needs head_dim 64 or 128");
  TTMI_REQUIRE(q_pitch >= heads * d && out_pitch >= heads * d, "rows overlap: a pitch is too small");
  TTMI_REQUIRE(dtype == TTMI_F32 || dtype == TTMI_F16 || dtype == TTMI_BF16, "unsupported dtype");
  TTMI_REQUIRE(sight->window >= 0 && max_tokens >= 0 && max_length >= 0, "window, max_tokens and max_length must not be negative");
  TTMI_REQUIRE(batch->tokens * heads < 1 << 30 && 2 * batch->batch * cache->kv_heads < 1 << 23, "more rows or sequences than one launch takes");
  const float scale_log2e = scale * 1.4426950408889634f;
  TTMI_REQUIRE(scale > 0.f && scale_log2e <= std::numeric_limits<float>::max(), "scale must be positive, and finite times log2(e)");
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  TTMI_REQUIRE(q != nullptr && out != nullptr, "q or out is null");
  TTMI_REQUIRE(rows_aligned(q, q_pitch, dtype) && rows_aligned(out, out_pitch, dtype), "rows of q and out must be 16-byte aligned");
  TTMI_REQUIRE((reinterpret_cast<uintptr_t>(sight->families) & 3) == 0, "families is not aligned to its elements");
  a.q = q, a.out = out, a.keys = cache->keys, a.values = cache->values, a.q_pitch = q_pitch, a.out_pitch = out_pitch;
  a.heads = (int)heads, a.group = (int)(heads / cache->kv_heads), a.causal = causal != 0;
  a.window = (int)std::min<int64_t>(sight->window, 1 << 30);
  a.scale_log2e = scale_log2e;
  const int sinks = (int)std::min<int64_t>(sight->sinks, 1 << 30);
  TTMI_DISPATCH_FLOAT(dtype, T, {
    const dim3 grid(a.view.tokens, a.heads);
    if (d == 64) hipLaunchKernelGGL((sight_kernel<T, 64>), grid, dim3(64), 0, static_cast<hipStream_t>(stream), a, sinks);
    else hipLaunchKernelGGL((sight_kernel<T, 128>), grid, dim3(64), 0, static_cast<hipStream_t>(stream), a, sinks);
  });
  return launch_status("paged_attention_sight");
}

}  // extern "C"
