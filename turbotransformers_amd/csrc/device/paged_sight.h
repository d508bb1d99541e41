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

// How a.shares workgroups are divided.  Work on a family is counted in steps of 64 keys of a block of 128 rows, that on the others in rounds of the few-rows kernel.  What a step costs a workgroup, in
// sixteenths of a microsecond with two workgroups on a CU, and what a round does where all of them read: its bytes at 9.8 GB/s.
template <typename T, int D>
constexpr int kStepCost = sizeof(T) == 4 ? (D == 128 ? 200 : 120) : (D == 128 ? 88 : 64);
template <typename T, int D>
constexpr int kRoundCost = 16 * kRound * 2 * D * (int)sizeof(T) / 9800;
struct Shares {
  int steps;          // of a part of a family's keys, at most
  int items;          // parts of blocks of rows of all families, for one key/value head
  int family_groups;  // workgroups that take them, for one head
  int few_groups;     // and those that are left for sequences with few rows
};
struct FamilyWork {  // of a lane's family
  int blocks, steps;
};
__device__ __forceinline__ FamilyWork family_work(const PagedArgs& a, const LaneSequences& lanes) {
  return {(int)(((int64_t)lanes.family_tokens * a.group + kTileRows - 1) / kTileRows), lanes.family_keys / 64};
}
__device__ __forceinline__ int family_parts(int steps, int most) { return (steps + most - 1) / most; }
// For kernels that follow, behind the partial results.
struct ShareNote {
  int steps, few_groups;
  int64_t units;
};
template <int D>
__device__ __forceinline__ ShareNote* share_note(const PagedArgs& a) {
  return reinterpret_cast<ShareNote*>(a.partial + a.rows * (D + 2));
}
// walk, *units: those of the few-rows kernel (and the first 64 sequences, where there are no more).
template <typename T, int D>
__device__ __forceinline__ Shares shares_of(const PagedArgs& a, Walk& walk, int64_t* units) {
  const int kv_heads = a.view.kv_heads;
  const bool few = a.run_few && a.few_splits > 0, single = a.view.batch <= kWave;
  *units = 0;
  if (few) *units = count_units<true>(a, walk);
  else if (single) walk.lanes = lane_sequences(a, 0);
  // (sums of 64 numbers that are capped for the balance alone)
  constexpr int kCap = 1 << 24;
  int64_t steps = 0;
  int longest = 0;
  for (int base = 0; base < a.view.batch; base += kWave) {
    const FamilyWork w = family_work(a, single ? walk.lanes : lane_sequences(a, base));
    steps += sum_of_lanes((int)min((int64_t)w.blocks * w.steps, (int64_t)kCap));
    for (uint64_t more = __ballot(w.steps > longest); more != 0; more = __ballot(w.steps > longest))
      longest = __builtin_amdgcn_readlane(w.steps, __ffsll((unsigned long long)more) - 1);
  }
  Shares s;
  // (in floats: every workgroup finds the same, and those that follow are told)
  const float family_cost = (float)(steps * kv_heads) * kStepCost<T, D>, cost = family_cost + (float)*units * kRoundCost<T, D>;
  const float groups = fmaxf((float)kv_heads, cost > 0.f ? a.shares * (family_cost / cost) : 0.f);
  s.steps = max(max(a.family_least, (longest + a.family_splits - 1) / a.family_splits), (int)fminf(__builtin_ceilf((float)(steps * kv_heads) / groups), 0x1p30f));
  s.items = 0;
  for (int base = 0; base < a.view.batch; base += kWave) {
    const FamilyWork w = family_work(a, single ? walk.lanes : lane_sequences(a, base));
    s.items += sum_of_lanes(w.blocks * family_parts(w.steps, s.steps));
  }
  // (at least an eighth is left for the others)
  s.family_groups = min(s.items, max(1, (few ? a.shares - a.shares / 8 : a.shares) / kv_heads));
  s.few_groups = max(1, min(a.few_splits, a.shares - s.family_groups * kv_heads));
  return s;
}

// The item-th part of a block of a family's rows -> whether there is one.
struct Job {
  int b, block, part, chunk;
  Sequence seq;
  Family family;
};
__device__ __forceinline__ bool find_family_job(const PagedArgs& a, const Shares& s, int item, bool there, LaneSequences& lanes, Job* job) {
  int passed = 0;
  for (int base = 0; base < a.view.batch; base += kWave) {
    if (!there) lanes = lane_sequences(a, base);
    const FamilyWork w = family_work(a, lanes);
    const int mine = w.blocks * family_parts(w.steps, s.steps), upto = passed + sum_up_to_here(mine), all = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (item >= all) {
      passed = all;
      continue;
    }
    const int found = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(item < upto)) - 1);
    const int at = item - __builtin_amdgcn_readlane(upto - mine, found), blocks = __builtin_amdgcn_readlane(w.blocks, found);
    const int steps = __builtin_amdgcn_readlane(w.steps, found), parts = family_parts(steps, s.steps);
    // (workgroups beside each other have the same keys of a head, on one XCD where there are eight heads)
    job->b = base + found, job->part = at / blocks, job->block = at - job->part * blocks, job->chunk = (steps + parts - 1) / parts * 64;
    job->seq = lanes.family_sequence(found), job->family = lanes.family(found);
    return true;
  }
  return false;
}
// The share of a workgroup in the families' keys (`lanes`: the first 64 sequences, where there are no more), taken in turns where there are more than workgroups; or a part of a block of a sequence
// with many rows, over its own keys.
template <typename T, int D, bool SMALL, bool FAMILIES>
__device__ __forceinline__ void sight_tiles(const PagedArgs& a, bool families, const Shares& s, int group, LaneSequences lanes, TilesShared<T, D>& shared) {
  const int kv_heads = a.view.kv_heads, kv_head = group % kv_heads;
  if constexpr (!FAMILIES) {
    int b, block;
    if (!find_block(a, group / kv_heads / a.splits, &b, &block)) return;
    tiles<T, D, SMALL, true, false>(a, b, block, sequence(a, b), LaneSequences{}, Family{}, 0, kv_head, group / kv_heads % a.splits, shared);
    return;
  }
  const int step = families ? s.family_groups : 1, stop = families ? s.items : 1;
  bool there = a.view.batch <= kWave;
  for (int item = families ? group / kv_heads : 0; item < stop; item += step) {
    Job job;
    if (families) {
      if (!find_family_job(a, s, item, there, lanes, &job)) return;
    } else {
      if (!find_block(a, group / kv_heads / a.splits, &job.b, &job.block)) return;
      lanes = lane_sequences(a, job.b & ~(kWave - 1));
      job.part = group / kv_heads % a.splits, job.chunk = 0, job.seq = lanes.sequence(job.b % kWave), job.family = Family{};
    }
    there = false;  // (they are not kept where the registers are needed)
    tiles<T, D, SMALL, true, FAMILIES>(a, job.b, job.block, job.seq, lanes, job.family, job.chunk, kv_head, job.part, shared);
    if (item + step >= stop) break;  // (without waiting for what was stored)
    __syncthreads();
  }
}

// One launch: a.shares workgroups (FAMILIES) for families and for sequences with few rows, a.tile_groups for those with many, the rest, if any, for few rows (FEW).  So a
// CU has workgroups that multiply beside others that read.  (Families take registers and FEW does not cost any, but instructions: a prompt of 8192 tokens in a window of 1024, 32 and 8
// heads of 128, 206 us with both, 195 without.)
template <typename T, int D, bool SMALL, bool FAMILIES, bool FEW>
__global__ __launch_bounds__(256, 2) void sight_kernel(const PagedArgs a) {
  static_assert(!FEW || !SMALL, "with small pages sequences with few rows have a launch of their own");
  __shared__ union {
    TilesShared<T, D> tiles;
    FewRowsShared<T, D, 4> few;
  } shared;
  int group = blockIdx.x, few_groups = a.few_splits;
  Walk walk{};
  Shares s{};
  int64_t units = -1;
  const int shares = FAMILIES ? a.shares : 0;
  bool families = false, own = !FEW;
  if (FAMILIES && group < shares) {
    s = shares_of<T, D>(a, walk, &units);
    if (group == 0 && threadIdx.x == 0) *share_note<D>(a) = {s.steps, s.few_groups, units};
    families = group < s.family_groups * a.view.kv_heads;
    if (!families) group -= s.family_groups * a.view.kv_heads, few_groups = s.few_groups;
    if (!families && (!FEW || units == 0 || group >= few_groups)) return;
  } else {
    group -= shares;
    own = !FEW || group < a.tile_groups;
    if (!own) group -= a.tile_groups;
  }
  if (families || own) sight_tiles<T, D, SMALL, FAMILIES>(a, families, s, group, walk.lanes, shared.tiles);
  else if constexpr (FEW) few_rows<T, D, 4, false, true>(a, group, few_groups, walk, units, shared.few);
}

// A wavefront a row and head.
template <typename T, int D>
__global__ __launch_bounds__(256) void join_sight_kernel(const PagedArgs a) {
  const PagedView& view = a.view;
  const int row = blockIdx.x, head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (head >= a.heads) return;
  ShareNote note{};
  if (a.families != nullptr) note = *share_note<D>(a);
  // the row's sequence: the first that ends behind it
  Walk walk{};
  int b = -1;
  for (int base = 0; base < view.batch; base += kWave) {
    walk.lanes = lane_sequences(a, base);
    const int before = __popcll(__ballot(base + (int)(threadIdx.x % kWave) < view.batch && walk.lanes.ends <= row));
    if (before == kWave) continue;
    b = base + before;
    break;
  }
  if (b < 0 || b >= view.batch) return;
  const Sequence seq = walk.lanes.sequence(b - walk.lanes.base);
  if (row < seq.start || row >= seq.start + seq.tokens) return;
  const int kv_head = head / a.group, r = (row - seq.start) * a.group + head % a.group, rows = seq.tokens * a.group;
  const int64_t at = (int64_t)row * a.heads + head;
  int of_family = 0;
  if (seq.base > 0) {  // (as many parts as there are chunks, which are equal but for the last)
    const int steps = seq.base / 64, parts = family_parts(steps, note.steps), chunk = (steps + parts - 1) / parts;
    of_family = (steps + chunk - 1) / chunk;
  }
  int parts = 1;                    // of the sequence's own keys
  int64_t place = a.whole_at + at;  // of them, and how far they lie apart
  int64_t second = 0, step = 0;
  if (!a.run_few || (rows > kFewRows && !a.few_every)) {
    const Reach mine = seq.own_reach(a, row - seq.start);
    const int row0 = r / kTileRows * kTileRows, last = min(rows, row0 + kTileRows) - 1;
    const Span span = span_of<kSpanTiles<T>>(sight_of(seq.own_reach(a, row0 / a.group), seq.own_reach(a, last / a.group)), seq.base);
    parts = own_parts(mine, span, seq.base, seq.span_chunk(a));
    place = a.own_at + at * a.splits, second = place + 1, step = 1;
  } else if (a.families == nullptr) {
    return;
  } else if (a.few_splits > 0) {
    int64_t units = note.units;
    if (view.batch <= kWave) walk.base = 0, walk.before = 0, walk.rounds = rounds_of<true>(a, own_sequence(walk.lanes)),
                             walk.upto = (int64_t)sum_up_to_here(walk.rounds) * view.kv_heads;
    else units = count_units<true>(a, walk);
    const Sharers shared = sharers_of<true>(a, walk, units, sharers(view.page_shift >= 4 ? note.few_groups : a.few_splits, units), b, kv_head);
    if (shared.last > shared.first) {
      parts = (int)(shared.last - shared.first) + 1;
      place = (2 * shared.first + 1) * kFewRows + r, second = 2 * (shared.first + 1) * kFewRows + r, step = 2 * kFewRows;
    }
  }
  if (of_family == 0 && parts == 1) return;  // (there already)
  const int64_t family_place = a.family_at + at * a.family_splits;
  const int all = of_family + parts;
  const bool sees = seq.reach(a, row - seq.start).end > 0;
  T* const out = static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)head * D;
  const float* const ml = a.partial + a.rows * D;
  auto place_of = [&](int p) {
    const int own = p - of_family;
    return own < 0 ? family_place + p : own == 0 ? place : second + (own - 1) * step;
  };
  if (all > kWave) {
    join_parts_by_wavefront<T, D>(a.partial, ml, all, sees, place_of, out);
    return;
  }
  // up to 64 parts: each lane has what one weighs, and the sums, four columns a lane and a few parts at a time, are asked for without waiting for that
  constexpr int kThreads = D / 4, kBeside = kWave / kThreads, kAsked = 8;
  const int lane = (int)(threadIdx.x % kWave), d0 = lane % kThreads * 4, share = lane / kThreads;
  const int64_t mine = place_of(min(lane, all - 1));
  const floatx2 met = *reinterpret_cast<const floatx2*>(ml + 2 * mine);
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  float weight = 0.f, total = 0.f;
  for (int first = 0; first < all; first += kAsked * kBeside) {
    floatx4 x[kAsked];
#pragma unroll
    for (int i = 0; i < kAsked; ++i) {
      const int p = min(first + i * kBeside + share, all - 1);
      x[i] = *reinterpret_cast<const floatx4*>(a.partial + place_of(p) * D + d0);
    }
    if (first == 0) {
      const float best = group_max<kWave>(lane < all ? met[0] : -INFINITY);
      weight = lane < all ? __builtin_amdgcn_exp2f(met[0] - (best == -INFINITY ? 0.f : best)) : 0.f;
      total = group_sum<kWave>(lane < all ? met[1] * weight : 0.f);
    }
#pragma unroll
    for (int i = 0; i < kAsked; ++i) {
      const int p = first + i * kBeside + share;
      const float w = __shfl(weight, min(p, kWave - 1), kWave);
      if (p < all) sum += x[i] * w;
    }
  }
#pragma unroll
  for (int d = kThreads; d < kWave; d *= 2)
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] += __shfl_xor(sum[c], d, kWave);
  if (share != 0) return;
  const float inv = inverse_sum(total, sees);
  Vec<T, 4> y;
#pragma unroll
  for (int c = 0; c < 4; ++c) y.v[c] = from_float<T>(sum[c] * inv);
  store_vec<T, 4>(out + d0, y);
}

template <typename T>
void start_sight(const SightLaunch& l, int64_t head_dim, hipStream_t stream) {
  const PagedArgs& a = l.all;
  auto sized = [&](auto d) {
    constexpr int D = decltype(d)::value;
    const int shares = a.families != nullptr ? a.shares : 0;
    const bool small = a.view.page_shift < 4;
    // (where sequences with few rows are shared out among all workgroups, those are a.shares)
    const int few_groups = a.few_splits == 0 ? a.view.batch * a.view.kv_heads : shares > 0 ? 0 : a.few_splits;
    auto launch = [&](auto kernel, int groups) { hipLaunchKernelGGL(kernel, dim3(groups), dim3(256), 0, stream, a); };
    if (!l.run_tiles) start_few_rows<T, true>(l.few, head_dim, stream);
    else if (!small && a.run_few) {
      if (shares > 0) launch(sight_kernel<T, D, false, true, true>, shares + a.tile_groups + few_groups);
      else launch(sight_kernel<T, D, false, false, true>, a.tile_groups + few_groups);
      start_join_few_rows<T, D, true>(l.few, stream);
    } else {
      if (small && shares > 0) launch(sight_kernel<T, D, true, true, false>, shares + a.tile_groups);
      else if (small) launch(sight_kernel<T, D, true, false, false>, a.tile_groups);
      else if (shares > 0) launch(sight_kernel<T, D, false, true, false>, shares + a.tile_groups);
      else launch(sight_kernel<T, D, false, false, false>, a.tile_groups);
      if (a.run_few) start_few_rows<T, true>(l.few, head_dim, stream);
    }
    if (a.families != nullptr || (l.run_tiles && a.splits > 1))
      hipLaunchKernelGGL((join_sight_kernel<T, D>), dim3(a.view.tokens, (unsigned)ceil_div(a.heads, 4)), dim3(256), 0, stream, a);
  };
  if (head_dim == 64) sized(std::integral_constant<int, 64>{});
  else sized(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace ttmi
