// The operators over a decoder's keys and values in pages, on tensors: ttmi_rotary_append[_normed], ttmi_paged_attention[_sight] and ttmi_copy_pages with the
// checks of their arguments.  They are enqueued on the stream that is given, whatever the context's stream is, and share nothing between
// calls, so calls on different streams may overlap.  No counterpart in the reference.
#pragma once

#include <cstdint>
#include <functional>
#include <vector>

#include "core/tensor.h"

namespace turbo_transformers {
namespace layers {

// A tensor as an operator reads it: where it lies and how, not who owns it.
struct TensorView {
  static constexpr int kMostDims = 8;
  void* data = nullptr;
  DLDataType dtype{};
  DLDevice device{};
  int n_dim = 0;
  int64_t shape[kMostDims] = {}, stride[kMostDims] = {};

  TensorView() = default;
  explicit TensorView(const DLTensor& t);
  explicit TensorView(const core::Tensor& t);
  int64_t numel() const;
  bool IsDense(int from_dim = 0) const;  // whether dimensions from_dim, ... lie densely behind each other
};

// table int32 [batch, pages of a sequence], starts int32 [batch + 1], lengths int32 [batch]
struct PagedBatchViews {
  TensorView table, starts, lengths;
};

// Weights of the norms of queries and keys, [d] or [heads, d] of float32 or the tensors' type; either may be missing.
struct HeadNorms {
  const TensorView *q = nullptr, *k = nullptr;
  float eps = 1e-6f;
};

// What tokens see and what sequences share: ttmi_paged_sight, the families int32 [batch, 3] or null.
struct PagedSight {
  int64_t window = 0, sinks = 0;
  const TensorView* families = nullptr;
  int64_t family_count = 0, max_shared = 0;
};

namespace kernels {

// qkv [tokens, (heads + 2 kv_heads) * d] or [tokens, heads + 2 kv_heads, d], rows any distance apart; keys, values [pages, kv_heads, page_size, d];
// inv_freq float64 [rotary_dim / 2] or null; q_out [tokens, heads * d] or [tokens, heads, d], rows any distance apart.
void RotaryAppend(const TensorView& qkv, const TensorView& keys, const TensorView& values, const PagedBatchViews& batch, const TensorView* inv_freq,
                  bool interleaved, float amplitude, const HeadNorms& norms, const TensorView& q_out, int device, void* stream);
// q, out [tokens, heads * d] or [tokens, heads, d], rows any distance apart.  scale null: 1 / sqrt(d).  `workspace` gives device memory of as many
// bytes that stays until the call's work on the stream is done.
void PagedAttention(const TensorView& q, const TensorView& keys, const TensorView& values, const PagedBatchViews& batch, const TensorView& out,
                    int64_t max_tokens, int64_t max_length, const float* scale, bool causal, const PagedSight& sight,
                    const std::function<void*(int64_t)>& workspace, int device, void* stream);
// keys, values [pages, ...] or, of several layers, [layers, pages, kv_heads, page_size, d]
void CopyPages(const TensorView& keys, const TensorView& values, const std::vector<int32_t>& sources, const std::vector<int32_t>& destinations,
               int device, void* stream);

}  // namespace kernels
}  // namespace layers
}  // namespace turbo_transformers
