// Attention over pages where tokens see the first keys of their sequence besides a window, and where sequences share keys: the kernels of paged_few_rows.h and paged_tiles.h
// that know of both, in one launch, and what joins the results of a row.
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

// How a.shares workgroups are divided.  Work on a family's blocks of 128 rows is counted in steps of 64 keys of one, all other in rounds of the few-rows kernel.  What a round costs a workgroup, in
// sixteenths of a microsecond, where all of them read: its bytes at 9.8 GB/s.  What a step does beside them is measured (a tile is asked for one ahead, and comes late): us for 64 sequences behind
// 6000 common keys, bf16, 32 and 8 heads of 128, up to 1500 of their own, at 20 / 40 / 60 / 88 / 120 / 160: 67.5 / 48.9 / 43.8 / 43.5 / 44.8 / 49.4; fp16 of 64, 1000: 31.2 / 28.8 / 30.5 / 32.3 / 35.6 /
// 35.4; fp32 of 64, 600: 125 / 76.6 / 67.0 / 59.3 / 57.1 / 54.9; fp32 of 128, behind 4000, 300, at 120 / 220 / 300: 105 / 87.8 / 82.3.
template <typename T, int D>
constexpr int kStepCost = sizeof(T) == 4 ? (D == 128 ? 320 : 140) : (D == 128 ? 72 : 48);
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
  const int blocks = family_blocks(a, lanes).many;
  return {blocks, blocks > 0 ? lanes.family_keys / 64 : 0};
}
__device__ __forceinline__ int family_parts(int steps, int most) { return (steps + most - 1) / most; }
// For the kernel that follows, behind the partial results: the units of the few-rows kernel, how they are shared out, and how many come before each sequence.
struct ShareNote {
  int steps, few_groups;
  int64_t units;
};
template <int D>
__device__ __forceinline__ ShareNote* share_note(const PagedArgs& a) {
  return reinterpret_cast<ShareNote*>(a.partial + a.rows * (D + 2));
}
template <int D>
__device__ __forceinline__ int64_t* units_before(const PagedArgs& a) {
  return reinterpret_cast<int64_t*>(share_note<D>(a) + 1);
}
// A part of a block of a family's rows, or of a sequence's with many.
struct Job {
  int b, block, part, chunk;
  Sequence seq;
  Family family;
};
// The item-th of all, in parts of `steps` at most, which is among 64 sequences, `passed` items being those of others before.
__device__ __forceinline__ void family_job(const PagedArgs& a, const LaneSequences& lanes, int steps, int item, int passed, Job* job) {
  const FamilyWork w = family_work(a, lanes);
  const int mine = w.blocks * family_parts(w.steps, steps), upto = passed + sum_up_to_here(mine);
  const int lane = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(item < upto)) - 1);
  const int at = item - __builtin_amdgcn_readlane(upto - mine, lane), blocks = __builtin_amdgcn_readlane(w.blocks, lane);
  const int all = __builtin_amdgcn_readlane(w.steps, lane), parts = family_parts(all, steps);
  // (workgroups beside each other have the same keys of a head, on one XCD where there are eight heads)
  job->b = lanes.base + lane, job->part = at / blocks, job->block = at - job->part * blocks, job->chunk = (all + parts - 1) / parts * 64;
  job->seq = lanes.family_sequence(lane), job->family = lanes.family(lane);
}
// Up to kSeen times 64 sequences are asked for at once, and what is needed of them stays in registers until the workgroup knows its share; more are read again for each number.
constexpr int kSeen = 4;
// What a workgroup of a.shares finds out.
template <typename T, int D>
struct Scan {
  FamilyWork work[kSeen];
  int rounds[kSeen];
  Shares s;
  int64_t units;
};
__device__ __forceinline__ bool seen_at_once(const PagedArgs& a) { return a.view.batch <= kSeen * kWave; }
__device__ __forceinline__ bool few_shared(const PagedArgs& a) { return a.run_few && a.few_splits > 0; }
// f(number of the first, work of this lane's family) for 64 sequences after the other
template <typename T, int D, typename F>
__device__ __forceinline__ void each_family(const PagedArgs& a, const Scan<T, D>& scan, F f) {
  if (seen_at_once(a)) {
#pragma unroll
    for (int g = 0; g < kSeen; ++g)
      if (g * kWave < a.view.batch) f(g * kWave, scan.work[g]);
  } else {
    for (int base = 0; base < a.view.batch; base += kWave) f(base, family_work(a, lane_sequences(a, base)));
  }
}
template <typename T, int D>
__device__ __forceinline__ Scan<T, D> scan_of(const PagedArgs& a, Walk& walk) {
  const int kv_heads = a.view.kv_heads;
  Scan<T, D> scan;
  scan.units = 0;
  if (seen_at_once(a)) {
    LaneNumbers numbers[kSeen];
#pragma unroll
    for (int g = 0; g < kSeen; ++g)
      if (g * kWave < a.view.batch) numbers[g] = lane_numbers(a, g * kWave);
#pragma unroll
    for (int g = 0; g < kSeen; ++g) {
      scan.rounds[g] = 0, scan.work[g] = {0, 0};
      if (g * kWave < a.view.batch) {
        const LaneSequences lanes = lane_sequences(a, g * kWave, numbers[g]);
        scan.work[g] = family_work(a, lanes);
        if (g == 0) walk.lanes = lanes;
        if (few_shared(a)) {
          scan.rounds[g] = all_rounds_of(a, lanes);
          scan.units += (int64_t)sum_of_lanes(scan.rounds[g]) * kv_heads;
        }
      }
    }
  } else if (few_shared(a)) scan.units = count_units<kFamilies>(a, walk);
  // (sums of 64 numbers that are capped for the balance alone)
  constexpr int kCap = 1 << 24;
  int64_t steps = 0;
  int longest = 0;
  each_family(a, scan, [&](int, const FamilyWork& w) {
    steps += sum_of_lanes((int)min((int64_t)w.blocks * w.steps, (int64_t)kCap));
    for (uint64_t more = __ballot(w.steps > longest); more != 0; more = __ballot(w.steps > longest))
      longest = __builtin_amdgcn_readlane(w.steps, __ffsll((unsigned long long)more) - 1);
  });
  // (in floats: every workgroup finds the same, and the kernel that follows is told)
  Shares& s = scan.s;
  const float family_cost = (float)(steps * kv_heads) * kStepCost<T, D>, cost = family_cost + (float)scan.units * kRoundCost<T, D>;
  const float groups = fmaxf((float)kv_heads, cost > 0.f ? a.shares * (family_cost / cost) : 0.f);
  s.steps = max(max(a.family_least, (longest + a.family_splits - 1) / a.family_splits), (int)fminf(__builtin_ceilf((float)(steps * kv_heads) / groups), 0x1p30f));
  s.items = 0;
  each_family(a, scan, [&](int, const FamilyWork& w) { s.items += sum_of_lanes(w.blocks * family_parts(w.steps, s.steps)); });
  // (at least an eighth is left for the others)
  s.family_groups = min(s.items, max(1, (few_shared(a) ? a.shares - a.shares / 8 : a.shares) / kv_heads));
  s.few_groups = max(1, min(a.few_splits, a.shares - s.family_groups * kv_heads));
  return scan;
}
// One workgroup does, before it turns to its share.
template <typename T, int D>
__device__ __forceinline__ void tell(const PagedArgs& a, const Scan<T, D>& scan) {
  const int lane = (int)threadIdx.x;
  if (lane >= kWave) return;
  if (lane == 0) *share_note<D>(a) = {scan.s.steps, scan.s.few_groups, scan.units};
  int64_t before = 0;
  for (int base = 0; few_shared(a) && base < a.view.batch; base += kWave) {
    const int mine = all_rounds_of(a, lane_sequences(a, base)), upto = sum_up_to_here(mine);
    if (base + lane < a.view.batch) units_before<D>(a)[base + lane] = before + (int64_t)(upto - mine) * a.view.kv_heads;
    before += (int64_t)__builtin_amdgcn_readlane(upto, kWave - 1) * a.view.kv_heads;
  }
}
// The walk of the few-rows kernel where its workgroup begins.
template <typename T, int D>
__device__ __forceinline__ void begin_walk(const PagedArgs& a, const Scan<T, D>& scan, int workgroup, Walk& walk) {
  if (!seen_at_once(a)) return;
  const int64_t unit = quotient(scan.units * workgroup, sharers(scan.s.few_groups, scan.units));
  int64_t from = 0, before = 0;
  int base = 0;
#pragma unroll
  for (int g = 0; g < kSeen; ++g)
    if (g * kWave < a.view.batch) {
      if (before <= unit) base = g * kWave, from = before;
      before += (int64_t)sum_of_lanes(scan.rounds[g]) * a.view.kv_heads;
    }
  walk.ahead = true, walk.base = base, walk.before = from;
  if (base > 0) walk.lanes = lane_sequences(a, base);
  take_lanes(a, walk);
}

// The part of its block that a workgroup takes.  Workgroups go round the eight XCDs and the four quarters of each, and of a block's parts the last ones often have nothing to do: so the first part is
// another one from block to block, or one quarter would have most of the work (fp32, 3 prompts of 300 tokens, 8 heads of 128, four parts: 45.4 / 29.2 us).
__device__ __forceinline__ int part_of(const PagedArgs& a, int n) {
  const int block = n / a.splits;
  return (n % a.splits + (a.splits == 2 ? block / 2 : block)) % a.splits;
}

// One launch: a.shares workgroups (FAMILIES) for families and for sequences with few rows, a.tile_groups for those with many, the rest, if any, for few rows (FEW).  So a
// CU has workgroups that multiply beside others that read.  (Families take registers and FEW does not cost any, but instructions: a prompt of 8192 tokens in a window of 1024, 32 and 8
// heads of 128, 206 us with both, 195 without.)
// Heads of 128 in three parts each take the registers of two workgroups, which families and sequences with few rows cannot spare.
template <typename T, int D, bool FAMILIES, bool FEW>
constexpr bool kThirds = sizeof(T) == 4 && (D == 64 || (!FAMILIES && !FEW));
// A part of a block of rows, in three parts a number if they hold it.
template <typename T, int D, bool SMALL, bool FAMILIES, bool THIRDS, typename Shared>
__device__ __forceinline__ void part_of_block(const PagedArgs& a, const Job& job, LaneSequences lanes, int kv_head, Shared& shared) {
  int thread = threadIdx.x;
  if constexpr (THIRDS) {
    if (__builtin_expect(tiles<T, D, SMALL, true, FAMILIES, true>(a, job.b, job.block, job.seq, lanes, job.family, job.chunk, kv_head, job.part, thread, shared.tiles), 1)) return;
    __syncthreads();
    // (what both ways find out alike must not stay in registers meanwhile: the compiler is not to know that it is alike)
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(thread));
#endif
    if constexpr (FAMILIES) lanes = lane_sequences(a, __builtin_amdgcn_readfirstlane(lanes.base));
  }
  tiles<T, D, SMALL, true, FAMILIES, false>(a, job.b, job.block, job.seq, lanes, job.family, job.chunk, kv_head, job.part, thread, shared.whole);
}
template <typename T, int D, bool SMALL, bool FAMILIES, bool FEW>
__global__ __launch_bounds__(256, (D == 128 && kThirds<T, D, FAMILIES, FEW> ? 1 : 2)) void sight_kernel(const PagedArgs a) {
  static_assert(!FEW || !SMALL, "with small pages sequences with few rows have a launch of their own");
  __shared__ union {
    TilesShared<T, D, kThirds<T, D, FAMILIES, FEW>> tiles;
    TilesShared<T, D, false> whole;
    FewRowsShared<T, D, 4> few;
  } shared;
  const int kv_heads = a.view.kv_heads;
  int group = blockIdx.x;
  if constexpr (!FAMILIES) {
    if (!FEW || group < a.tile_groups) {
      Job job{};
      if (!find_block(a, group / kv_heads / a.splits, &job.b, &job.block)) return;
      job.part = part_of(a, group / kv_heads), job.seq = sequence(a, job.b);
      part_of_block<T, D, SMALL, false, kThirds<T, D, FAMILIES, FEW>>(a, job, LaneSequences{}, group % kv_heads, shared);
    } else if constexpr (FEW) {
      Walk walk{};
      few_rows<T, D, 4, false, kSinks>(a, group - a.tile_groups, a.few_splits, walk, -1, shared.few);
    }
  } else {
    Job job;
    LaneSequences lanes;
    int item = 0, step = 1, stop = 1, steps = 1;  // parts of families are taken in turns where there are more than workgroups
    int few_groups = -1;
    Walk walk{};
    int64_t units = -1;
    int base = 0, passed = 0;
    bool own = false;
    if (group < a.shares) {
      const Scan<T, D> scan = scan_of<T, D>(a, walk);
      if (group == 0) tell(a, scan);
      const int family_groups = scan.s.family_groups * kv_heads;
      if (group < family_groups) {
        item = group / kv_heads, step = scan.s.family_groups, stop = scan.s.items, steps = scan.s.steps;
        int upto = 0;
        each_family(a, scan, [&](int from, const FamilyWork& w) {
          if (upto <= item) base = from, passed = upto;
          upto += sum_of_lanes(w.blocks * family_parts(w.steps, steps));
        });
        lanes = walk.lanes;
        if (base > 0 || !seen_at_once(a)) lanes = lane_sequences(a, base);
      } else {
        group -= family_groups, few_groups = scan.s.few_groups, units = scan.units;
        if (!FEW || units == 0 || group >= few_groups) return;
        begin_walk(a, scan, group, walk);
      }
    } else {
      group -= a.shares;
      own = group < a.tile_groups;
      if (!own) group -= a.tile_groups, few_groups = 0;
    }
    if (few_groups >= 0) {
      if constexpr (FEW) few_rows<T, D, 4, false, kFamilies>(a, group, few_groups, walk, units, shared.few);
      return;
    }
    for (;;) {
      if (own) {
        if (!find_block(a, group / kv_heads / a.splits, &job.b, &job.block)) return;
        lanes = lane_sequences(a, job.b & ~(kWave - 1));
        job.part = part_of(a, group / kv_heads), job.chunk = 0, job.seq = lanes.sequence(job.b % kWave), job.family = Family{};
      } else family_job(a, lanes, steps, item, passed, &job);
      part_of_block<T, D, SMALL, true, kThirds<T, D, FAMILIES, FEW>>(a, job, lanes, group % kv_heads, shared);
      item += step;
      if (item >= stop) break;
      __syncthreads();
      // on to the 64 sequences that have it
      for (;;) {
        if (base >= a.view.batch) return;
        lanes = lane_sequences(a, base);  // (not kept meanwhile: the registers are needed)
        const FamilyWork w = family_work(a, lanes);
        const int upto = passed + sum_of_lanes(w.blocks * family_parts(w.steps, steps));
        if (item < upto) break;
        passed = upto, base += kWave;
      }
    }
  }
}

// A wavefront a row and head, or (MANY) several heads.
template <typename T, int D, bool MANY>
__global__ __launch_bounds__(256) void join_sight_kernel(const PagedArgs a) {
  const PagedView& view = a.view;
  const int row = blockIdx.x, first_head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (first_head >= a.heads) return;
  ShareNote note{};
  if (a.families != nullptr) note = *share_note<D>(a);
  // the row's sequence: the first that ends behind it
  const int lane = (int)(threadIdx.x % kWave);
  LaneSequences lanes;
  int b = 0;
  int64_t before = 0;
  // (among the last 64 of which the first begins up to it: two trips to memory.  256 sequences, one token each, 32 heads of 128: 15.4 us for one after the other, 13.0 so, 11.6 with more heads a wavefront.)
  int base = 0;
  if (view.batch > kWave)
    for (int from = 0; from < view.batch; from += kWave * kWave) {
      const int at = from + lane * kWave;
      const int begun = __popcll(__ballot(at < view.batch && view.starts[min(at, view.batch - 1)] <= row));
      if (begun == 0) break;
      base = from + (begun - 1) * kWave;
    }
  if (a.families != nullptr && a.run_few && a.few_splits > 0) before = units_before<D>(a)[min(base + lane, view.batch - 1)];
  lanes = lane_sequences(a, base);
  b = base + __popcll(__ballot(base + lane < view.batch && lanes.ends <= row));
  if (b >= min(view.batch, base + kWave)) return;
  const Sequence seq = lanes.sequence(b - lanes.base);
  const int64_t before_all = before;
  // (the family that it leads comes first)
  before = lane_of(before, b - lanes.base);
  if (a.families != nullptr) {
    const int blocks = family_blocks(a, lanes).few;
    before += (int64_t)__builtin_amdgcn_readlane(blocks * family_rounds_of(lanes, blocks), b - lanes.base) * view.kv_heads;
  }
  if (row < seq.start || row >= seq.start + seq.tokens) return;
  // its family's parts: how many, or where they begin
  const int rows = seq.tokens * a.group;
  int family_parts_all = 0, family_start = 0;
  int64_t family_before = 0;
  if (seq.base > 0) {
    const int leader = __builtin_amdgcn_readlane(lanes.leader, b - lanes.base);
    LaneSequences theirs = lanes;
    if (leader < lanes.base) theirs = lane_sequences(a, leader & ~(kWave - 1));
    if (__builtin_amdgcn_readlane(family_blocks(a, theirs).few, leader - theirs.base) == 0) {  // (as many parts as there are chunks, which are equal but for the last)
      const int steps = seq.base / 64, most = family_parts(steps, note.steps), chunk = (steps + most - 1) / most;
      family_parts_all = (steps + chunk - 1) / chunk;
    } else {
      family_start = __builtin_amdgcn_readlane(theirs.start, leader - theirs.base);
      family_before = leader < lanes.base ? units_before<D>(a)[leader] : lane_of(before_all, leader - lanes.base);
    }
  }
  const bool by_tiles = !a.run_few || (rows > kFewRows && !a.few_every), sees = seq.reach(a, row - seq.start).end > 0;
  if (!by_tiles && a.families == nullptr) return;
  const int rounds = !by_tiles && a.few_splits > 0 ? rounds_of<true>(a, seq) : 0;
  const int64_t workgroups = a.families != nullptr ? sharers(view.page_shift >= 4 ? note.few_groups : a.few_splits, note.units) : 0;
  const float* const ml = a.partial + a.rows * D;
  for (int head = first_head; head < (MANY ? a.heads : first_head + 1); head += MANY ? 4 * gridDim.y : 1) {
    const int kv_head = head / a.group, r = (row - seq.start) * a.group + head % a.group;
    const int64_t at = (int64_t)row * a.heads + head;
    // parts of what it has in common with its family, and of its own: where the first is, and how far the others lie apart behind the second
    int of_family = 0;
    int64_t family_place = a.family_at + at * a.family_splits, family_second = family_place + 1, family_step = 1;
    if (seq.base > 0) {
      of_family = max(1, family_parts_all);
      if (family_parts_all == 0) {
        const int of_rows = (row - family_start) * a.group + head % a.group, block = of_rows / kFewRows, family_rounds = kStart + seq.base / kRound;
        const Sharers shared = sharers_of(family_before + (int64_t)(block * view.kv_heads + kv_head) * family_rounds, family_rounds, note.units, workgroups);
        if (shared.last > shared.first) {
          of_family = (int)(shared.last - shared.first) + 1;
          family_place = (2 * shared.first + 1) * kFewRows + of_rows % kFewRows;
          family_second = 2 * (shared.first + 1) * kFewRows + of_rows % kFewRows, family_step = 2 * kFewRows;
        }
      }
    }
    int parts = 1;                    // of the sequence's own keys
    int64_t place = a.whole_at + at;  // of them, and how far they lie apart
    int64_t second = 0, step = 0;
    if (by_tiles) {
      const Reach mine = seq.own_reach(a, row - seq.start);
      const int row0 = r / kTileRows * kTileRows, last = min(rows, row0 + kTileRows) - 1;
      const Span span = span_of<kSpanTiles<T>>(sight_of(seq.own_reach(a, row0 / a.group), seq.own_reach(a, last / a.group)), seq.base);
      parts = own_parts(mine, span, seq.base, seq.span_chunk(a));
      place = a.own_at + at * a.splits, second = place + 1, step = 1;
    } else if (a.few_splits > 0) {
      const Sharers shared = sharers_of(before + (int64_t)rounds * kv_head, rounds, note.units, workgroups);
      if (shared.last > shared.first) {
        parts = (int)(shared.last - shared.first) + 1;
        place = (2 * shared.first + 1) * kFewRows + r, second = 2 * (shared.first + 1) * kFewRows + r, step = 2 * kFewRows;
      }
    }
    if (of_family == 0 && parts == 1) continue;  // (there already)
    const int all = of_family + parts;
    T* const out = static_cast<T*>(a.out) + (int64_t)row * a.out_pitch + (int64_t)head * D;
    auto place_of = [&](int p) {
      const int own = p - of_family;
      if (own < 0) return p == 0 ? family_place : family_second + (p - 1) * family_step;
      return own == 0 ? place : second + (own - 1) * step;
    };
    if (all > kWave) {
      join_parts_by_wavefront<T, D>(a.partial, ml, all, sees, place_of, out);
      continue;
    }
    // up to 64 parts: each lane has what one weighs, and the sums, four columns a lane and a few parts at a time, are asked for without waiting for that
    constexpr int kThreads = D / 4, kBeside = kWave / kThreads, kAsked = 8;
    const int d0 = lane % kThreads * 4, share = lane / kThreads;
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
    if (share == 0) {
      const float inv = inverse_sum(total, sees);
      Vec<T, 4> y;
#pragma unroll
      for (int c = 0; c < 4; ++c) y.v[c] = from_float<T>(sum[c] * inv);
      store_vec<T, 4>(out + d0, y);
    }
  }
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
    if (!l.run_tiles) start_few_rows<T, kSinks>(l.few, head_dim, stream);
    else if (!small && a.run_few) {
      if (shares > 0) launch(sight_kernel<T, D, false, true, true>, shares + a.tile_groups + few_groups);
      else launch(sight_kernel<T, D, false, false, true>, a.tile_groups + few_groups);
      if (shares == 0) start_join_few_rows<T, D, kSinks>(l.few, stream);
    } else {
      if (small && shares > 0) launch(sight_kernel<T, D, true, true, false>, shares + a.tile_groups);
      else if (small) launch(sight_kernel<T, D, true, false, false>, a.tile_groups);
      else if (shares > 0) launch(sight_kernel<T, D, false, true, false>, shares + a.tile_groups);
      else launch(sight_kernel<T, D, false, false, false>, a.tile_groups);
      if (a.run_few && shares > 0) start_few_rows<T, kFamilies>(l.few, head_dim, stream);
      else if (a.run_few) start_few_rows<T, kSinks>(l.few, head_dim, stream);
    }
    // (as many heads a wavefront as leave four workgroups a CU: each finds out first what its row's sequence is)
    const int64_t fours = ceil_div(a.heads, 4), per = std::max<int64_t>(1, std::min<int64_t>(fours, (int64_t)a.view.tokens * fours / (4 * compute_units())));
    auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.view.tokens, (unsigned)ceil_div(fours, per)), dim3(256), 0, stream, a); };
    if (a.families != nullptr || (l.run_tiles && a.splits > 1)) {
      if (per > 1) join(join_sight_kernel<T, D, true>);
      else join(join_sight_kernel<T, D, false>);
    }
  };
  if (head_dim == 64) sized(std::integral_constant<int, 64>{});
  else sized(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace ttmi
