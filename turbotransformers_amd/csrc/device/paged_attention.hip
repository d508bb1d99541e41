// Attention of new tokens over keys and values in pages: o = sum_j p_j v_j with p = softmax_j(scale q . k_j) over the keys that a token sees.
// One pass over the keys: with the maximum m and the sum l of exp(s_j - m) so far, a tile of new scores moves m to m', scales what was summed by
// exp(m - m') and adds its own exp(s_j - m') and exp(s_j - m') v_j.  All of it in fp32.
#include "paged.h"

namespace ttmi {

// One wavefront per token and head: a lane per key for the scores, a lane per column for the sum over the values.
template <typename T, int D>
__global__ __launch_bounds__(64) void paged_attention_kernel(const T* __restrict__ q, int64_t q_pitch, T* __restrict__ out, int64_t out_pitch, int group,
                                                             const T* __restrict__ keys, const T* __restrict__ values, const PagedView view, float scale,
                                                             int causal, int64_t window) {
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int b = sequence_of(view, token);
  if (b >= view.batch || token < view.starts[b]) return;
  const int64_t held = view.table_pitch << view.page_shift;
  const int length = (int)min((int64_t)view.lengths[b], held), position = view.lengths[b] - view.starts[b + 1] + token;
  if (length < view.lengths[b] && lane == 0) page_error(view);
  const int end = causal ? min(length, position + 1) : length;
  const int begin = window > 0 ? (int)max((int64_t)0, (int64_t)position - window + 1) : 0;
  __shared__ float q_lds[D], p_lds[64];
  __shared__ int64_t row_lds[64];
  for (int i = lane; i < D; i += 64) q_lds[i] = to_float(q[token * q_pitch + (int64_t)head * D + i]) * scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[D / 64] = {};
  for (int j0 = begin; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY;
    int64_t row = 0;
    if (j < end) {
      int page = view.table[(int64_t)b * view.table_pitch + (j >> view.page_shift)];
      if ((unsigned)page >= (unsigned)view.pages) {
        page_error(view);
        page = 0;
      }
      row = ((((int64_t)page * view.kv_heads + head / group) << view.page_shift) + (j & ((1 << view.page_shift) - 1))) * D;
      s = 0.f;
      constexpr int W = 16 / (int)sizeof(T);
      for (int i = 0; i < D; i += W) {
        const Vec<T, W> k = load_vec<T, W>(keys + row + i);
#pragma unroll
        for (int e = 0; e < W; ++e) s += to_float(k.v[e]) * q_lds[i + e];
      }
    }
    const float top = fmaxf(m, group_max<64>(s));
    const float shrink = m == -INFINITY ? 0.f : expf(m - top), p = s == -INFINITY ? 0.f : expf(s - top);
    l = l * shrink + group_sum<64>(p);
    m = top;
    p_lds[lane] = p, row_lds[lane] = row;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] *= shrink;
    for (int i = 0; i < min(64, end - j0); ++i)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) acc[c] += p_lds[i] * to_float(values[row_lds[i] + c * 64 + lane]);
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) out[token * out_pitch + (int64_t)head * D + c * 64 + lane] = from_float<T>(acc[c] * inv);
}

}  // namespace ttmi

using namespace ttmi;

extern "C" {

int ttmi_paged_attention_workspace(const ttmi_paged_cache* cache, const ttmi_paged_batch* batch, int64_t heads, int64_t max_tokens, int64_t max_length,
                                   int64_t window, int dtype, int64_t* bytes) {
  PagedView view;
  TTMI_REQUIRE(bytes != nullptr, "bytes is null");
  if (int rc = paged_view(cache, batch, heads, &view)) return rc;
  *bytes = 0;
  return 0;
}

int ttmi_paged_attention(const void* q, int64_t q_pitch, void* out, int64_t out_pitch, int64_t heads, const ttmi_paged_cache* cache,
                         const ttmi_paged_batch* batch, int64_t max_tokens, int64_t max_length, float scale, int causal, int64_t window,
                         void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  PagedView view;
  if (int rc = paged_view(cache, batch, heads, &view)) return rc;
  const int64_t d = cache->head_dim;
  TTMI_REQUIRE(d == 64 || d == 128, "paged attention needs head_dim 64 or 128");
  TTMI_REQUIRE(q_pitch >= heads * d && out_pitch >= heads * d, "rows overlap: a pitch is too small");
  TTMI_REQUIRE(dtype == TTMI_F32 || dtype == TTMI_F16 || dtype == TTMI_BF16, "unsupported dtype");
  TTMI_REQUIRE(window >= 0 && max_tokens >= 0 && max_length >= 0, "window, max_tokens and max_length must not be negative");
  TTMI_REQUIRE(scale > 0.f && scale <= 3e38f, "scale must be positive and finite");
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  TTMI_REQUIRE(q != nullptr && out != nullptr, "q or out is null");
  TTMI_REQUIRE(rows_aligned(q, q_pitch, dtype) && rows_aligned(out, out_pitch, dtype), "rows of q and out must be 16-byte aligned");
  TTMI_DISPATCH_FLOAT(dtype, T, {
    const dim3 grid((unsigned)view.tokens, (unsigned)heads);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(64), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(q), q_pitch, static_cast<T*>(out), out_pitch,
                         (int)(heads / cache->kv_heads), static_cast<const T*>(cache->keys), static_cast<const T*>(cache->values), view, scale, causal, window);
    };
    if (d == 64) launch(paged_attention_kernel<T, 64>);
    else launch(paged_attention_kernel<T, 128>);
  });
  return launch_status("paged_attention");
}

}  // extern "C"
