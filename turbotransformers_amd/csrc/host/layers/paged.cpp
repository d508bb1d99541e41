#include "layers/paged.h"

#include <cmath>

#include "core/enforce.h"
#include "ttmi.h"

namespace turbo_transformers {
namespace layers {

TensorView::TensorView(const DLTensor& t) : dtype(t.dtype), device(t.device), n_dim(t.ndim) {
  TT_ENFORCE(t.ndim <= kMostDims, "a tensor has more than %d dimensions", kMostDims);
  data = t.data == nullptr ? nullptr : static_cast<char*>(t.data) + t.byte_offset;
  int64_t dense = 1;
  for (int i = n_dim - 1; i >= 0; --i) {
    shape[i] = t.shape[i];
    stride[i] = t.strides != nullptr ? t.strides[i] : dense;
    dense *= t.shape[i];
  }
}

TensorView::TensorView(const core::Tensor& t) : dtype(t.dtype()), device(t.device_ctx()), n_dim((int)t.n_dim()) {
  TT_ENFORCE(n_dim <= kMostDims, "a tensor has more than %d dimensions", kMostDims);
  data = const_cast<void*>(t.raw());
  int64_t dense = 1;
  for (int i = n_dim - 1; i >= 0; --i) {
    shape[i] = t.shape(i);
    stride[i] = dense;
    dense *= shape[i];
  }
}

int64_t TensorView::numel() const {
  int64_t n = 1;
  for (int i = 0; i < n_dim; ++i) n *= shape[i];
  return n;
}

bool TensorView::IsDense(int from_dim) const {
  int64_t dense = 1;
  for (int i = n_dim - 1; i >= from_dim; --i) {
    if (shape[i] != 1 && stride[i] != dense) return false;
    dense *= shape[i];
  }
  return true;
}

namespace kernels {
namespace {

void RequireOn(const TensorView& t, int device, const char* what) {
  if (!core::IsGpu(t.device.device_type)) TT_THROW("%s: tensor is not on the GPU; this build has no CPU kernels", what);
  TT_ENFORCE(t.device.device_id == device, "%s: the tensor is on device %d, the current device is %d", what, (int)t.device.device_id, device);
}

int FloatType(const TensorView& t, const char* what) {
  const int type = core::ToDeviceDType(t.dtype);
  TT_ENFORCE(type == TTMI_F32 || type == TTMI_F16 || type == TTMI_BF16, "%s: expected float32, float16 or bfloat16", what);
  return type;
}

void RequireInts(const TensorView& t, int n_dim, int device, const char* what) {
  RequireOn(t, device, what);
  TT_ENFORCE(core::ToDeviceDType(t.dtype) == TTMI_I32, "%s: expected int32", what);
  TT_ENFORCE(t.n_dim == n_dim && (t.numel() == 0 || t.IsDense()), "%s: expected a dense tensor of %d dimensions", what, n_dim);
}

struct CacheArgs {
  ttmi_paged_cache cache;
  int type;
};
CacheArgs Cache(const TensorView& keys, const TensorView& values, int device) {
  for (const TensorView* t : {&keys, &values}) {
    RequireOn(*t, device, "keys and values");
    TT_ENFORCE(t->n_dim == 4 && (t->numel() == 0 || t->IsDense()), "keys and values must be dense, [pages, kv_heads, page_size, head_dim]");
  }
  for (int i = 0; i < 4; ++i) TT_ENFORCE_EQ(keys.shape[i], values.shape[i], "keys and values differ in shape");
  TT_ENFORCE(core::SameDataType(keys.dtype, values.dtype), "keys and values differ in type");
  CacheArgs out;
  out.type = FloatType(keys, "keys and values");
  out.cache = {keys.data, values.data, keys.shape[0], keys.shape[1], keys.shape[2], keys.shape[3]};
  return out;
}

ttmi_paged_batch Batch(const PagedBatchViews& batch, int64_t tokens, int device) {
  RequireInts(batch.table, 2, device, "table");
  RequireInts(batch.starts, 1, device, "starts");
  RequireInts(batch.lengths, 1, device, "lengths");
  const int64_t n = batch.lengths.shape[0];
  TT_ENFORCE(batch.table.shape[0] == n && batch.starts.shape[0] == n + 1, "table, starts and lengths differ in their number of sequences");
  return {static_cast<const int32_t*>(batch.table.data), batch.table.shape[1], static_cast<const int32_t*>(batch.starts.data),
          static_cast<const int32_t*>(batch.lengths.data), n, tokens};
}

// Rows of heads of d elements, [tokens, heads * d] or [tokens, heads, d]: how many heads, and how far rows are apart.
struct RowArgs {
  int64_t heads, pitch;
};
RowArgs Rows(const TensorView& t, const CacheArgs& cache, int device, const char* what) {
  RequireOn(t, device, what);
  TT_ENFORCE(core::ToDeviceDType(t.dtype) == cache.type, "%s: the type is not that of the cache", what);
  const int64_t d = cache.cache.head_dim;
  TT_ENFORCE((t.n_dim == 2 && d > 0 && t.shape[1] % d == 0) || (t.n_dim == 3 && t.shape[2] == d), "%s: expected [tokens, heads * head_dim] or [tokens, heads, head_dim]",
             what);
  TT_ENFORCE(t.numel() == 0 || t.IsDense(1), "%s: rows must be dense", what);
  const int64_t width = t.n_dim == 2 ? t.shape[1] : t.shape[1] * d;
  TT_ENFORCE(t.shape[0] <= 1 || t.stride[0] >= width, "%s: rows overlap", what);
  return {width / d, t.shape[0] > 1 ? t.stride[0] : width};
}

// Whether two sets of rows share an element: rows of one pitch may stand side by side.
bool Share(const TensorView& a, const RowArgs& a_rows, const TensorView& b, const RowArgs& b_rows, int64_t d) {
  const int64_t size = a.dtype.bits / 8, n = a.shape[0];
  if (n == 0) return false;
  const int64_t a_width = a_rows.heads * d * size, b_width = b_rows.heads * d * size, a_pitch = a_rows.pitch * size, b_pitch = b_rows.pitch * size;
  const intptr_t a0 = reinterpret_cast<intptr_t>(a.data), b0 = reinterpret_cast<intptr_t>(b.data);
  if (a0 + (n - 1) * a_pitch + a_width <= b0 || b0 + (n - 1) * b_pitch + b_width <= a0) return false;
  if (a_pitch != b_pitch) return true;
  const int64_t off = ((b0 - a0) % a_pitch + a_pitch) % a_pitch;  // of b's rows within a's
  return off < a_width || off + b_width > a_pitch;
}

// Whether rows, or one of two dense tensors, reach into the other's memory.
bool Meet(const TensorView& a, int64_t a_bytes, const TensorView& b, int64_t b_bytes) {
  const intptr_t a0 = reinterpret_cast<intptr_t>(a.data), b0 = reinterpret_cast<intptr_t>(b.data);
  return a_bytes > 0 && b_bytes > 0 && a0 < b0 + b_bytes && b0 < a0 + a_bytes;
}
int64_t Bytes(const TensorView& dense) { return dense.numel() * (dense.dtype.bits / 8); }
int64_t Bytes(const TensorView& t, const RowArgs& rows, int64_t d) {
  return t.shape[0] > 0 ? ((t.shape[0] - 1) * rows.pitch + rows.heads * d) * (t.dtype.bits / 8) : 0;
}

}  // namespace

void RotaryAppend(const TensorView& qkv, const TensorView& keys, const TensorView& values, const PagedBatchViews& batch, const TensorView* inv_freq,
                  bool interleaved, float amplitude, const TensorView& q_out, int device, void* stream) {
  const CacheArgs cache = Cache(keys, values, device);
  const RowArgs in = Rows(qkv, cache, device, "qkv");
  RowArgs out = Rows(q_out, cache, device, "queries");
  TT_ENFORCE(in.heads == out.heads + 2 * cache.cache.kv_heads && qkv.shape[0] == q_out.shape[0],
             "qkv must hold the queries' heads and twice the cache's, a row for each of the queries'");
  const bool in_place = q_out.data == qkv.data;
  if (in_place && qkv.shape[0] <= 1) out.pitch = in.pitch;  // (a single row has none of its own)
  TT_ENFORCE(in_place || !Share(qkv, in, q_out, out, cache.cache.head_dim), "the queries' place overlaps qkv");
  const int64_t held = Bytes(keys);
  TT_ENFORCE(!Meet(keys, held, values, held), "keys and values overlap");
  for (const TensorView* t : {&keys, &values}) {
    TT_ENFORCE(!Meet(*t, held, qkv, Bytes(qkv, in, cache.cache.head_dim)) && !Meet(*t, held, q_out, Bytes(q_out, out, cache.cache.head_dim)),
               "qkv or the queries' place overlaps the cache");
  }
  const ttmi_paged_batch args = Batch(batch, qkv.shape[0], device);
  int64_t rotary_dim = 0;
  if (inv_freq != nullptr) {
    RequireOn(*inv_freq, device, "inv_freq");
    TT_ENFORCE(inv_freq->dtype.code == kDLFloat && inv_freq->dtype.bits == 64 && inv_freq->n_dim == 1 && inv_freq->IsDense(),
               "inv_freq: expected a dense float64 tensor of one dimension");
    rotary_dim = 2 * inv_freq->shape[0];
  }
  TT_DEVICE_CALL(ttmi_rotary_append(qkv.data, in.pitch, q_out.data, out.pitch, out.heads, &cache.cache, &args,
                                    inv_freq != nullptr ? static_cast<const double*>(inv_freq->data) : nullptr, rotary_dim, interleaved ? 1 : 0, amplitude,
                                    cache.type, stream));
}

void PagedAttention(const TensorView& q, const TensorView& keys, const TensorView& values, const PagedBatchViews& batch, const TensorView& out,
                    int64_t max_tokens, int64_t max_length, const float* scale, bool causal, int64_t window,
                    const std::function<void*(int64_t)>& workspace, int device, void* stream) {
  const CacheArgs cache = Cache(keys, values, device);
  const RowArgs from = Rows(q, cache, device, "q"), to = Rows(out, cache, device, "out");
  TT_ENFORCE(from.heads == to.heads && q.shape[0] == out.shape[0], "q and out differ in shape");
  TT_ENFORCE(!Share(q, from, out, to, cache.cache.head_dim), "out overlaps q");
  for (const TensorView* t : {&keys, &values})
    TT_ENFORCE(!Meet(*t, Bytes(*t), out, Bytes(out, to, cache.cache.head_dim)), "out overlaps the cache");
  const ttmi_paged_batch args = Batch(batch, q.shape[0], device);
  const float factor = scale != nullptr ? *scale : (float)(1.0 / std::sqrt((double)cache.cache.head_dim));
  int64_t bytes = 0;
  TT_DEVICE_CALL(ttmi_paged_attention_workspace(&cache.cache, &args, from.heads, max_tokens, max_length, window, cache.type, &bytes));
  TT_DEVICE_CALL(ttmi_paged_attention(q.data, from.pitch, out.data, to.pitch, from.heads, &cache.cache, &args, max_tokens, max_length, factor, causal ? 1 : 0,
                                      window, bytes > 0 ? workspace(bytes) : nullptr, bytes, cache.type, stream));
}

void CopyPages(const TensorView& keys, const TensorView& values, const std::vector<int32_t>& sources, const std::vector<int32_t>& destinations, int device,
               void* stream) {
  for (const TensorView* t : {&keys, &values}) {
    RequireOn(*t, device, "keys and values");
    TT_ENFORCE((t->n_dim == 4 || t->n_dim == 5) && (t->numel() == 0 || t->IsDense()),
               "keys and values must be dense, [pages, kv_heads, page_size, head_dim] or [layers, pages, kv_heads, page_size, head_dim]");
  }
  TT_ENFORCE_EQ(keys.n_dim, values.n_dim, "keys and values differ in shape");
  for (int i = 0; i < keys.n_dim; ++i) TT_ENFORCE_EQ(keys.shape[i], values.shape[i], "keys and values differ in shape");
  TT_ENFORCE(core::SameDataType(keys.dtype, values.dtype), "keys and values differ in type");
  TT_ENFORCE(!Meet(keys, Bytes(keys), values, Bytes(values)), "keys and values overlap");
  TT_ENFORCE_EQ(sources.size(), destinations.size(), "one destination for each source");
  const bool many = keys.n_dim == 5;
  const int64_t layers = many ? keys.shape[0] : 1, pages = keys.shape[many ? 1 : 0];
  int64_t page_bytes = keys.dtype.bits / 8;
  for (int i = many ? 2 : 1; i < keys.n_dim; ++i) page_bytes *= keys.shape[i];
  TT_DEVICE_CALL(ttmi_copy_pages(keys.data, values.data, layers, pages, page_bytes, sources.data(), destinations.data(), (int64_t)sources.size(), stream));
}

}  // namespace kernels
}  // namespace layers
}  // namespace turbo_transformers
