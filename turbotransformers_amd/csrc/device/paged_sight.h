// Attention over pages where tokens see the first keys of their sequence besides a window, and where sequences share keys: the kernels of paged_few_rows.h and paged_tiles.h
// with SIGHT, and what joins the results of a row.
//
// With families a row's softmax is one over two lists of keys, its family's [0, P) and its sequence's own [P, length):
//     o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i,   m = max m_i,
// over the parts i that both were cut into, m_i the reference point, l_i the sum and o_i the weighted values of part i.  The rows of a family are those of all its sequences,
// so its keys are read once for 128 rows instead of once for each sequence, and the matrix instructions have full tiles where decoding alone would give them 4 of 16 rows.
#pragma once

#include "paged_few_rows.h"
#include "paged_tiles.h"

namespace ttmi {

namespace {

template <typename T, int D, bool SMALL>
__global__ __launch_bounds__(256, 2) void sight_tiles_kernel(const PagedArgs a, int own_blocks) {
  __shared__ TilesShared<T, D> shared;
  const int kv_heads = a.view.kv_heads, family_groups = a.families != nullptr ? kv_heads * a.family_blocks * a.family_splits : 0;
  const bool families = (int)blockIdx.x < family_groups;
  const int group = families ? blockIdx.x : blockIdx.x - family_groups, splits = families ? a.family_splits : a.splits;
  const int kv_head = group % kv_heads, part = group / kv_heads % splits;
  // (more blocks than was said are taken in turns)
  const int step = families ? a.family_blocks : own_blocks;
  for (int block = group / kv_heads / splits, upto = INT32_MAX; block < upto; block += step) {
    upto = tiles<T, D, SMALL, true>(a, block, kv_head, part, families, shared);
    __syncthreads();
  }
}

// A wavefront a row and head.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_sight_kernel(const PagedArgs a, const PagedArgs few, bool run_few) {
  const PagedView& view = a.view;
  const int row = blockIdx.x, b = sequence_of(view, row), head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (b >= view.batch || head >= a.heads) return;
  const Sequence seq = sequence_of_batch<true>(a, b);
  if (row < seq.start) return;
  const int kv_head = head / a.group, r = (row - seq.start) * a.group + head % a.group, rows = seq.tokens * a.group;
  const int64_t at = (int64_t)row * a.heads + head;
  int family_parts = 0;
  if (seq.base > 0) {
    Sequence family;
    family.length = seq.base;
    const int chunk = family_chunk(a, family);
    family_parts = (seq.base + chunk - 1) / chunk;
  }
  int parts = 1;                     // of the sequence's own keys
  int64_t place = few.whole_at + at;  // of them, and how far they lie apart
  int64_t second = 0, step = 0;
  if (!run_few || (rows > kFewRows && !few.every)) {
    const Reach mine = seq.own_reach(a, row - seq.start);
    const int row0 = r / kTileRows * kTileRows, last = min(rows, row0 + kTileRows) - 1;
    const Span span = span_of<kSpanTiles>(sight_of(seq.own_reach(a, row0 / a.group), seq.own_reach(a, last / a.group)), seq.base);
    parts = own_parts(mine, span, seq.base, seq.span_chunk(a));
    place = a.own_at + at * a.splits, second = place + 1, step = 1;
  } else if (a.families == nullptr) {
    return;
  } else if (few.splits > 0) {
    const Sharers shared = sharers_of<true>(few, b, kv_head);
    if (shared.last > shared.first) {
      parts = (int)(shared.last - shared.first) + 1;
      place = (2 * shared.first + 1) * kFewRows + r, second = 2 * (shared.first + 1) * kFewRows + r, step = 2 * kFewRows;
    }
  }
  if (family_parts == 0 && parts == 1) return;  // (there already)
  const int64_t family_place = a.family_at + at * a.family_splits;
  join_parts_by_wavefront<T, D>(
      a.partial, a.partial + a.rows * D, family_parts + parts, seq.reach(a, row - seq.start).end > 0,
      [&](int p) {
        const int own = p - family_parts;
        return own < 0 ? family_place + p : own == 0 ? place : second + (own - 1) * step;
      },
      static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)head * D);
}

template <typename T>
void start_sight(const SightLaunch& l, int64_t head_dim, hipStream_t stream) {
  const PagedArgs& a = l.tiles;
  auto sized = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (l.run_tiles) {
      const int64_t groups = (int64_t)a.view.kv_heads * ((a.families != nullptr ? (int64_t)a.family_blocks * a.family_splits : 0) + (int64_t)l.own_blocks * a.splits);
      if (a.view.page_shift < 4) hipLaunchKernelGGL((sight_tiles_kernel<T, D, true>), dim3((unsigned)groups), dim3(256), 0, stream, a, l.own_blocks);
      else hipLaunchKernelGGL((sight_tiles_kernel<T, D, false>), dim3((unsigned)groups), dim3(256), 0, stream, a, l.own_blocks);
    }
    if (l.run_few) start_few_rows<T, true>(l.few, head_dim, stream);
    if (a.families != nullptr || (l.run_tiles && a.splits > 1))
      hipLaunchKernelGGL((join_sight_kernel<T, D>), dim3(a.view.tokens, (unsigned)ceil_div(a.heads, 4)), dim3(256), 0, stream, a, l.few, l.run_few);
  };
  if (head_dim == 64) sized(std::integral_constant<int, 64>{});
  else sized(std::integral_constant<int, 128>{});
}

}  // namespace

}  // namespace ttmi
