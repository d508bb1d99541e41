// Attention of new tokens over keys and values in pages: o = sum_j p_j v_j with p = softmax_j(scale q . k_j) over the keys that a token sees.
// One pass over the keys: with the maximum m and the sum l of exp(s_j - m) so far, a tile of new scores moves m to m', scales what was summed by
// exp(m - m') and adds its own exp(s_j - m') and exp(s_j - m') v_j.  Scores, m, l and the sums in fp32; exp(x) as 2^(x log2 e).  In 16-bit types the probabilities are rounded to the type for the second product,
// which the matrix instructions take no wider, and l sums the rounded ones.
//
// Two kernels share a batch by the rows (new tokens times query heads of a key/value head) of its sequences: up to 16 of them paged_few_rows.hip, more
// paged_tiles.hip.  This file cuts the work: keys of a sequence into parts, where there are few rows and heads, whose results a small kernel joins.
#include "paged_attention.h"

#include <limits>

namespace ttmi {
namespace {

constexpr int64_t kWidest = 1 << 30;  // windows: no position lies beyond it

struct PagedPlan {
  bool few, tiles;  // which kernels run; one alone takes all sequences
  int few_rows, few_splits, few_waves, tile_chunk, tile_splits;
  int64_t few_floats, tile_floats;  // of the workspace
};

// Many rows, `units` blocks of them with up to `reach` keys: into parts of at least `least` keys, where it is two of them.  A workgroup alone on its CU is done a third earlier than one of two, so the
// parts are as many as the CUs hold one each, but where those would be long (five times the least and more), and a CU that has none idles long: then as many as make two.
// us, whole chip / twice that: bf16, 8 key heads of 64, a prompt of 1000 tokens 21.7 / 26.2, 400 tokens behind 1500 keys 27.0 / 27.4, behind 6000 58.0 / 51.8, 700 behind 6000
// 100.6 / 78.8; head_dim 128 30.4 / 41.1, 39.2 / 39.4, 81.8 / 75.0, 146 / 118.5.
void cut(int64_t units, int64_t least, int64_t reach, bool window, int* chunk, int* splits) {
  const int64_t most = reach < 2 * least ? 1 : ceil_div(reach, least), cus = compute_units();
  auto made = [&](int64_t workgroups) { return std::min(std::max<int64_t>(1, workgroups / std::max<int64_t>(1, units)), most); };
  int64_t parts = made(cus);
  if (reach >= 5 * least * parts) parts = made(2 * cus);
  const int64_t size = ceil_div(ceil_div(reach, parts), 64) * 64;
  *splits = parts > 1 ? (int)(ceil_div(reach, size) + (window ? 1 : 0)) : 1;
  *chunk = (int)size;
}

// Few rows: up to so many bytes of keys and values of one sequence and head are one workgroup's.  A CU fetches about 50 GB/s while few others read, so these take 6 us, what sharing them out
// and joining the parts costs besides their share.  Where the pairs fill the chip it is the launch to join that counts: 256 sequences of 620 keys, 8 key heads of 128, 115 / 126, 64 of 1 to 600 keys
// 18.0 / 24.7.  us a call, one workgroup / shared: bf16, head_dim 128, 8 sequences of 255 keys (130 KB) 7.2 / 12.4, 500 10.6 / 13.5,
// 1000 (512 KB) 15.6 / 15.9, 2000 25.2 / 22.6, 1 sequence of 1000 14.8 / 12.6; fp16, head_dim 64, 12 heads, 1 sequence of 1000 (256 KB) 9.7 / 12.1, 2000 14.4 / 12.1.
constexpr int64_t kWholeBytes = 320 << 10;

PagedPlan plan(const PagedView& view, int64_t heads, int64_t max_tokens, int64_t max_length, int64_t window, int dtype) {
  PagedPlan p;
  window = std::min(window, kWidest);
  const int64_t group = heads / view.kv_heads, tokens = view.tokens, batch = std::max(1, view.batch);
  const int64_t held = view.table_pitch << view.page_shift;
  const int64_t longest = std::max<int64_t>(1, max_length > 0 ? std::min(max_length, held) : held);
  const int64_t most = max_tokens > 0 ? std::min(max_tokens, tokens) : tokens;
  const int64_t reach = window > 0 ? std::min(longest, window + most) : longest;
  p.tiles = most * group > kFewRows;
  // One launch instead of two where sequences have many rows on average and none of them many keys: the kernel for many rows takes those with few as well (40 sequences decoding and 3
  // chunks of 200 to 900 tokens, 1000 keys seen: two launches 38.0 us, one 25.6).  Where one may have more than
  // 64 of its tiles, a workgroup would walk over them with a row or four of 128 alive, and sequences with few rows keep a kernel that cuts their keys, if there can be
  // any (the tokens would make so many sequences of the most only).
  // us, one launch / two, one key length for all decoding sequences (1000, 4000, 8000, 16000, 100000), chunks without keys before them:
  //   bf16, 32 and 8 heads of 128: 1 decoding, a chunk of 512     26.5 / 31.6,    43.2 / 36.0,   66.4 / 38.6,  115 / 46,   640 / 110
  //                                8, one of 2048                 63.1 / 77.8,    93.2 / 88.1,    166 / 108,   315 / 165, 1893 / 619
  //                                40, 3 of 500                   51.7 / 63.8,     139 / 160,     256 / 266,   495 / 492
  //   fp16, 16 and 4 heads of 64:  8, one of 2048                 36.3 / 45.9,    57.2 / 48.7,    105 / 53,    203 / 63,  1252 / 187
  //   fp32, 12 heads of 64:        8, one of 2048                  155 / 173,      309 / 193,     595 / 234,  1166 / 301, 7117 / 973  (2000: 168 / 180)
  // Sequences that all have many rows pay the launches of the other kernel: 6 chunks of 400 to 600 tokens behind up to 9000 keys 220 / 224.
  const int64_t long_walk = 64 * (dtype == TTMI_F32 ? 32 : 64);
  const bool some_few = most * batch > tokens;
  p.few = !p.tiles || tokens * group / batch < 64 || (reach > long_walk && some_few);
  p.few_rows = p.tiles ? kFewRows : (int)(most * group);
  p.few_splits = reach * 2 * view.head_dim * (int64_t)dtype_size(dtype) <= kWholeBytes ? 0 : 2 * compute_units();
  p.few_waves = p.few_splits == 0 && batch * view.kv_heads < compute_units() ? 8 : 4;
  // (The least that takes longer than joining: fp32, whose matrix instructions take sixteen times as long, us for one prompt of 200 tokens, 4 key heads of 64, parts of 256 / 64
  // at least 20.9 / 15.1; 16-bit types, 400 tokens, 8 key heads, parts of 512 / 256 / 128 11.9 / 14.3 / 15.7, 100 tokens behind 8000 keys, one key head, 17.1 / 15.0 / 16.6.)
  cut(view.kv_heads * (tokens * group / 128 + std::min(batch, tokens)), dtype == TTMI_F32 ? 64 : 256, reach, window > 0, &p.tile_chunk, &p.tile_splits);
  const int64_t d = view.head_dim;
  p.few_floats = p.few ? 2ll * p.few_splits * kFewRows * (d + 2) : 0;
  p.tile_floats = p.tiles && p.tile_splits > 1 ? tokens * heads * p.tile_splits * (d + 2) : 0;
  return p;
}

}  // namespace
}  // namespace ttmi

using namespace ttmi;

extern "C" {

int ttmi_paged_attention_workspace(const ttmi_paged_cache* cache, const ttmi_paged_batch* batch, int64_t heads, int64_t max_tokens, int64_t max_length,
                                   int64_t window, int dtype, int64_t* bytes) {
  PagedView view;
  TTMI_REQUIRE(bytes != nullptr, "bytes is null");
  if (int rc = paged_view(cache, batch, heads, &view)) return rc;
  TTMI_REQUIRE(window >= 0 && max_tokens >= 0 && max_length >= 0, "window, max_tokens and max_length must not be negative");
  *bytes = 0;
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  const PagedPlan p = plan(view, heads, max_tokens, max_length, window, dtype);
  *bytes = (p.few_floats + p.tile_floats) * 4;
  return 0;
}

int ttmi_paged_attention(const void* q, int64_t q_pitch, void* out, int64_t out_pitch, int64_t heads, const ttmi_paged_cache* cache,
                         const ttmi_paged_batch* batch, int64_t max_tokens, int64_t max_length, float scale, int causal, int64_t window,
                         void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  PagedArgs a;
  if (int rc = paged_view(cache, batch, heads, &a.view)) return rc;
  const int64_t d = cache->head_dim;
  TTMI_REQUIRE(d == 64 || d == 128, "paged attention needs head_dim 64 or 128");
  TTMI_REQUIRE(q_pitch >= heads * d && out_pitch >= heads * d, "rows overlap: a pitch is too small");
  TTMI_REQUIRE(dtype == TTMI_F32 || dtype == TTMI_F16 || dtype == TTMI_BF16, "unsupported dtype");
  TTMI_REQUIRE(window >= 0 && max_tokens >= 0 && max_length >= 0, "window, max_tokens and max_length must not be negative");
  // (a launch has less than 2^32 threads: 512 of them for a sequence and key/value head, or 256 for 128 rows besides)
  TTMI_REQUIRE(batch->tokens * heads < 1 << 30 && batch->batch * cache->kv_heads < 1 << 23, "more rows or sequences than one launch takes");
  const float scale_log2e = scale * 1.4426950408889634f;
  TTMI_REQUIRE(scale > 0.f && scale_log2e <= std::numeric_limits<float>::max(), "scale must be positive, and finite times log2(e)");
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  TTMI_REQUIRE(q != nullptr && out != nullptr, "q or out is null");
  TTMI_REQUIRE(rows_aligned(q, q_pitch, dtype) && rows_aligned(out, out_pitch, dtype), "rows of q and out must be 16-byte aligned");
  const PagedPlan p = plan(a.view, heads, max_tokens, max_length, window, dtype);
  const int64_t bytes = (p.few_floats + p.tile_floats) * 4;
  TTMI_REQUIRE(bytes == 0 || (workspace != nullptr && workspace_bytes >= bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "the workspace is too small or not 16-byte aligned");
  a.q = q, a.out = out, a.keys = cache->keys, a.values = cache->values, a.q_pitch = q_pitch, a.out_pitch = out_pitch;
  a.heads = (int)heads, a.group = (int)(heads / cache->kv_heads), a.causal = causal != 0;
  a.window = (int)std::min(window, kWidest);
  a.scale_log2e = scale_log2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.tiles) {
    a.every = !p.few, a.chunk = p.tile_chunk, a.splits = p.tile_splits;
    a.partial = static_cast<float*>(workspace) + p.few_floats;
    if (int rc = launch_tiles(a, dtype, d, s)) return rc;
  }
  if (p.few) {
    a.every = !p.tiles, a.few = p.few_rows, a.splits = p.few_splits, a.waves = p.few_waves;
    a.partial = static_cast<float*>(workspace);
    if (int rc = launch_few_rows(a, dtype, d, s)) return rc;
  }
  return 0;
}

}  // extern "C"
