// Attention of new tokens over keys and values in pages: o = sum_j p_j v_j with p = softmax_j(scale q . k_j) over the keys that a token sees.
// One pass over the keys: with the maximum m and the sum l of exp(s_j - m) so far, a tile of new scores moves m to m', scales what was summed by
// exp(m - m') and adds its own exp(s_j - m') and exp(s_j - m') v_j.  Scores, m, l and the sums in fp32; exp(x) as 2^(x log2 e).  In 16-bit types the probabilities are rounded to the type for the second product,
// which the matrix instructions take no wider, and l sums the rounded ones.
//
// Two kernels share a batch by the rows (new tokens times query heads of a key/value head) of its sequences: up to 16 of them paged_few_rows.hip, more
// paged_tiles.hip.  This file cuts the work: keys of a sequence into parts, where there are few rows and heads, whose results a small kernel joins.
#include "paged_attention.h"

#include <cmath>
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

// Blocks of 128 rows over `steps` steps of 64 keys, cut into how many parts, and about how long they take (us): workgroups of one part, two on a CU, in as many rounds as there are (a last one that
// leaves each CU at most one takes about half as long, but not where they wait for keys), and what writing and joining the parts costs.
struct Cut {
  int64_t parts;
  double us;
};
double rounds_of(double groups, bool single) {
  const double cus = compute_units(), rounds = std::floor(groups / (2 * cus)), rest = groups - rounds * 2 * cus;
  return rounds + (rest <= 0 ? 0 : rest <= cus && !single ? 0.55 : 1);
}
Cut best_cut(double blocks, int64_t steps, double step, bool single, int64_t tokens, int64_t heads, int64_t head_dim) {
  const double join = (double)tokens * heads * (head_dim + 2) * 8 / (single ? 9e6 : 4.5e6);
  Cut best = {1, 1e30};
  for (int64_t parts = 1; parts <= 64 && parts <= steps; ++parts) {
    const double us = rounds_of(blocks * parts, single) * (double)ceil_div(steps, parts) * step + parts * join;
    if (us < best.us) best = {parts, us};
  }
  return best;
}
// us a step where two workgroups are on a CU: bound by products, or (single tokens, few of whose rows are alive) by the wait for keys
double step_us(int dtype, int64_t head_dim, bool single) {
  if (dtype == TTMI_F32) return head_dim == 128 ? (single ? 20 : 27) : single ? 8 : 5.5;
  return head_dim == 128 ? (single ? 4 : 2.3) : (single ? 2.2 : 1.35);
}
bool single_tokens(const PagedView& view, int64_t heads) { return view.tokens * (heads / view.kv_heads) <= kFewRows * (int64_t)view.batch; }
// Rows of a family up to which the few-rows kernel takes its keys, 16 rows at a time, from memory or again from L2: the other reads them once for up to 128, but one wavefront of it computes 32 of
// them alone, which takes fp32 sixteen times as long.  us, one token each, 12 heads of 64 / 32 and 8 of 128, that kernel / this one: fp16, 16 families of 4 behind 8000 keys 105 / 84, 8 of 8 63 / 47; bf16, 4 rows
// a sequence, 16 of 4 161 / 115, 8 of 8 (32 rows) 72 / 92; fp32 16 of 4 412 / 156, 8 of 8 253 / 90, 64 (64 rows) behind 1000 39.5 / 29.0; 4 rows a sequence, 16 of 4 828 / 213, 16 (64 rows) behind
// 8000 81 / 58.
int family_few_rows(int dtype) { return dtype == TTMI_F32 ? 64 : 16; }
struct FamilyGuess {
  double count, blocks;  // of them, and of rows
  int64_t steps;  // of the longest
};
FamilyGuess guess_families(const PagedView& view, int64_t heads, const ttmi_paged_sight& sight) {
  const int64_t held = view.table_pitch << view.page_shift, shared = sight.max_shared > 0 ? std::min(sight.max_shared, held) : held;
  const int64_t count = std::max<int64_t>(1, std::min<int64_t>(sight.family_count, view.batch / 2));
  return {(double)count, (double)std::max(count, ceil_div(view.tokens * (heads / view.kv_heads), 128)), std::max<int64_t>(1, shared / 64)};
}

// With first keys that stay visible and with families.  The sequences' own keys are cut as ever (their number is guessed from max_length: a sequence on its own may be that long).  A family's are
// cut on the device, which knows how many there are; here it is said into how many parts at most, and how many workgroups there will be: one for each part, or two a CU where sequences
// with few rows take a share of them (16 questions about 20000 tokens, 32 and 8 heads of 128: 1 / 2 / 3 / 5 / 8 parts 650 / 570 / 498 / 475 / 487 us).
struct SightPlan {
  PagedPlan own;
  int shares, family_splits, family_least, family_few, own_blocks;
  int64_t few_rows, own_rows, family_rows, whole_rows, floats;  // of the workspace
};
PagedPlan plan_own(const PagedView& view, int64_t heads, int64_t max_tokens, int64_t max_length, const ttmi_paged_sight& sight, int dtype) {
  const int64_t sinks = std::min(sight.sinks, kWidest), window = sight.window > 0 ? std::min(std::min(sight.window, kWidest) + sinks + 128, kWidest) : 0;
  return plan(view, heads, max_tokens, max_length, window, dtype);
}
SightPlan plan_sight(const PagedView& view, int64_t heads, int64_t max_tokens, int64_t max_length, const ttmi_paged_sight& sight, int dtype) {
  SightPlan p;
  p.own = plan_own(view, heads, max_tokens, max_length, sight, dtype);
  const int64_t group = heads / view.kv_heads, tokens = view.tokens, d = view.head_dim;
  p.own_blocks = p.own.tiles ? (int)(tokens * group / 128 + std::min<int64_t>(view.batch, tokens)) : 0;
  p.shares = p.family_splits = p.family_least = p.family_few = 0, p.family_rows = p.whole_rows = 0;
  const bool families = sight.families != nullptr;
  if (families) {
    const FamilyGuess guess = guess_families(view, heads, sight);
    const bool single = single_tokens(view, heads);
    const int64_t two = 2 * compute_units(), pairs = (int64_t)guess.blocks * view.kv_heads;
    p.family_least = dtype == TTMI_F32 ? 1 : 2;
    if (p.own.few) p.own.few_splits = 2 * compute_units(), p.family_few = family_few_rows(dtype);
    // (single tokens: as many as the device may find best for all workgroups there are)
    const int64_t parts = single ? ceil_div(guess.steps, std::max<int64_t>(p.family_least, pairs * guess.steps / two)) + 1
                                 : best_cut((double)pairs, guess.steps, step_us(dtype, d, single), single, tokens, heads, d).parts;
    p.family_splits = (int)parts;
    // (not more than there is room for at a time, where these are all; each head has one, and leaves as many)
    const bool with_few = p.own.few && p.own.few_splits > 0;
    p.shares = (int)std::max<int64_t>(single ? two : with_few ? std::max(two, pairs * parts * 5 / 4) : pairs * parts, 2 * (int64_t)view.kv_heads);
    p.family_rows = tokens * heads * p.family_splits;
    p.whole_rows = p.own.few ? tokens * heads : 0;
  }
  p.few_rows = p.own.few ? 2ll * p.own.few_splits * kFewRows : 0;
  p.own_rows = p.own.tiles && (families || p.own.tile_splits > 1) ? tokens * heads * p.own.tile_splits : 0;
  p.floats = (p.few_rows + p.own_rows + p.family_rows + p.whole_rows) * (d + 2) + (families ? 4 + 2 * (int64_t)view.batch : 0);
  return p;
}

// Whether reading a family's keys once is worth it: a second launch, which joins what they give with what the sequences' own keys do, and blocks of 128 rows that may be mostly empty, for reads
// that the caches would take most of.  Both are estimated, with what fits the measured; us, families / none, one token each and 50 keys of its own, behind 1000, 2000, 4000, 8000 keys:
//   bf16, 32 and 8 heads of 128: 8 sequences 17.4 / 14.8, 18.6 / 16.6, 20.3 / 21.4, 25.3 / 29.5; 64 26.7 / 28.0, 30.0 / 45.1, 32.2 / 78.6, 40.7 / 147; 256 59.6 / 95.1 .. 68.9 / 297 (4000);
//                                8 families of 2 20.4 / 17.5 .. 51.6 / 53.9; 4 of 8 21.9 / 21.5, 26.6 / 31.1, 30.0 / 48.7, 39.8 / 82.3; 16 of 4 30.7 / 29.3, 37.7 / 47.5, 54.8 / 88.7, 115 / 180
//   fp16, 12 heads of 64:        16 sequences 15.0 / 9.0, 15.0 / 18.5, 14.6 / 25.0, 18.3 / 36.6; 16 families of 4 26.3 / 20.4, 31.7 / 40.6, 45.1 / 65.9, 81.8 / 137
//   fp32, the same heads:        4 sequences 15.8 / 12.8, 15.9 / 15.7, 16.1 / 21.3, 22.3 / 27.5; 64 28.1 / 46.8 .. 49.3 / 262; 32 and 8 heads of 128, 64: 59.7 / 55.5, 63.3 / 92.0 .. 141 / 319
// Where the two are within some per cent of each other it may take the slower one: over 195 such batches what it takes is 0.3 % slower on average than the better of the two, at most 8 % where it shares
// (8 families of 8 behind 512 keys, fp32 25.7 / 23.9) and 16 where it does not (2 sequences behind 4000, fp32 16.1 / 18.7), none alone 46 %.
//
// Of more tokens a sequence (more than 16 rows a key/value head on average) all blocks are the kernel's for many rows: what counts is the longest part of one (`step` for each of its steps of 64 keys),
// what all blocks do (`work` for as many steps of a full block as there are workgroups at a time, of which each 32 rows take most), partial results written and joined (`join`, for 10^6 bytes of them both
// ways), and with families a second set of blocks, for the sequences' own keys (`block`, for as many as there are at a time).  us, families / none, bf16, 32 and 8 heads of 128:
//   32 sequences of 20 tokens behind 1000, 2000, 4000 keys 57 / 30, 71 / 49, 89 / 88; 8 families of 4 79 / 31, 74 / 50, 104 / 88; 16 of 50 behind 2000, 5000 83 / 52, 124 / 112; 100 of 6 behind 2000, 4000 99 / 117 (no), 114 / 194
//   fp32: 8 families of 4 with 50 tokens behind 700, 2000 347 / 226, 657 / 553 (yes); heads of 64, 12 of them: 4 of 50 behind 2000 41 / 56, 48 of 20 behind 700 81 / 138
// Over 714 batches of 5 to 150 tokens a sequence what it takes is 1.1 % slower on average than the better of the two, at most 31 % (16 of 150 behind 2000, fp32 843 / 1101, no), none alone 19 %; over 122 random batches of all kinds 0.3 and 19 %.
//
// Windows: common keys that they hide are estimated as half of seen ones (many tokens: a quarter).  us, families / none, behind 8000 keys, windows of 500, 1500 and 4000 with 4 first tokens: bf16, 32 and 8
// heads of 128, 64 sequences 34.7 / 16.3, 36.6 / 38.5, 37.9 / 79.4; 16 families of 4 58.5 / 17.4, 60.2 / 39.8, 71.7 / 89.6; 64 with 20 tokens each 108 / 47.6, 123 / 69.6, 175 / 145; fp32, 16 families of 4
// 99.2 / 38.3, 107 / 81.4, 159 / 193.  Over 400 such batches what it takes is 1.7 % slower on average than the better of the two, at most 57 % (16 of 20 tokens, fp32, window 4000, 270 / 424, no), none alone
// 29 %.
struct ManyTokens {
  double once, step, work, join, block;  // us
};
bool many_tokens_share(const PagedView& view, int64_t heads, int64_t max_length, const ttmi_paged_sight& sight, int dtype, const PagedPlan& own, const FamilyGuess& guess, int64_t walked) {
  const bool f32 = dtype == TTMI_F32, wide = view.head_dim == 128;
  ManyTokens a = f32 ? (wide ? ManyTokens{17, 4.9, 16.5, 0.17, 0} : ManyTokens{15.5, 0.8, 13, 0, 0}) : wide ? ManyTokens{14.5, 0.55, 2.1, 0.16, 0} : ManyTokens{12, 0.4, 1.5, 0.2, 0};
  const ManyTokens s = f32 ? (wide ? ManyTokens{27, 4.5, 14.7, 0.6, 38} : ManyTokens{20, 1.1, 5.3, 0.45, 35}) : wide ? ManyTokens{17.5, 0.45, 1.8, 0.35, 22} : ManyTokens{13, 0.4, 1.1, 0.55, 18};
  // (behind a gap fp32 by three parts a number, which heads of 128 have without families and sequences of few rows)
  if (f32 && sight.window > 0 && sight.sinks > 0 && !(wide && own.few)) a.step *= 0.65, a.work *= 0.65;
  const int64_t held = view.table_pitch << view.page_shift, longest = max_length > 0 ? std::min(max_length, held) : held, shared = std::min(sight.max_shared, held);
  const double rows = (double)view.tokens * (double)(heads / view.kv_heads), batch = view.batch, at_a_time = 2.0 * compute_units() / (double)view.kv_heads;
  const double own_steps = std::max(1.0, (double)std::min(longest - shared, sight.window > 0 ? sight.window : kWidest) / 64);
  // (half a block, or half of 32 rows, of each sequence is empty, and each has one)
  const double blocks = std::max(batch, rows / 128 + batch / 2), full = 0.7 * std::max(batch, rows / 32 + batch / 2) / 4 + 0.3 * blocks;
  const double family_full = 0.7 * std::max(guess.count, std::ceil(rows / 32)) / 4 + 0.3 * guess.blocks;
  const double join = (double)view.tokens * (double)heads * (double)(view.head_dim + 2) * 8e-6, steps = (double)guess.steps;
  const int64_t parts = best_cut(guess.blocks * (double)view.kv_heads, walked, step_us(dtype, view.head_dim, false), false, view.tokens, heads, view.head_dim).parts;
  const double alone = a.once + a.step * std::min((double)ceil_div(own.tile_chunk, 64), steps + own_steps) + a.work * full * (steps + own_steps) / at_a_time +
                       (own.tile_splits > 1 ? a.join * join * own.tile_splits : 0);
  const double together = s.once + s.step * (double)ceil_div(walked, parts) + s.work * (family_full * (double)walked + full * own_steps) / at_a_time + s.join * join * (double)(parts + 1) +
                          s.block * blocks / at_a_time;
  return together < alone;
}

// Where nothing is known they are taken as they come.
bool sharing_pays(const PagedView& view, int64_t heads, int64_t max_tokens, int64_t max_length, const ttmi_paged_sight& sight, int dtype) {
  if (sight.families == nullptr) return false;
  if (sight.family_count == 0 || sight.max_shared == 0) return true;
  FamilyGuess guess = guess_families(view, heads, sight);
  const int64_t all = guess.steps;
  if (sight.window > 0) guess.steps = std::min(all, ceil_div(std::min(sight.window, kWidest) + std::min(sight.sinks, kWidest), 64) + 1);  // (seen of the common keys)
  const PagedPlan own = plan_own(view, heads, max_tokens, max_length, sight, dtype);
  const bool f32 = dtype == TTMI_F32, wide = view.head_dim == 128, single = single_tokens(view, heads);
  const double step = step_us(dtype, view.head_dim, single), rows = (double)view.tokens * (double)(heads / view.kv_heads), batch = view.batch;
  const double bytes = guess.steps * 64.0 * (2 * view.kv_heads * view.head_dim * (double)dtype_size(dtype));
  // Common keys that a window hides: they are cut into parts with the others, of which the ends alone are trimmed, so they cost those who share some of what they would if they were seen.
  const int64_t walked = guess.steps + (all - guess.steps) / (single ? 2 : 4);
  if (!single) return many_tokens_share(view, heads, max_length, sight, dtype, own, guess, walked);
  // each by itself: the common keys again and again, out of the caches, and a launch that joins
  double alone = (own.few && own.few_splits == 0 ? 7 : f32 ? (wide ? 14 : 13.5) : 12) + batch * bytes / (f32 ? 12.5e6 : 15e6);
  if (own.tiles) alone += 5;
  if (alone <= 11) return false;  // (what a second launch and the rest of it take at least)
  // shared: as many bytes as families read, or blocks of their rows over parts of the keys
  const double count = (double)std::min<int64_t>(sight.family_count, std::max(1, view.batch / 2)), most = std::ceil(rows / count);
  double shared;
  if (most <= family_few_rows(dtype)) shared = (f32 ? (wide ? 16 : 14.5) : 13) + 0.05 * batch + count * std::ceil(most / kFewRows) * bytes * ((double)walked / (double)guess.steps) / 6e6;
  else shared = (f32 ? (wide ? 22 : 12) : (wide ? 12 : 11)) + (f32 ? 0.15 : 0.1) * batch +
                best_cut(guess.blocks * (double)view.kv_heads, walked, step, single, view.tokens, heads, view.head_dim).us;
  return shared < alone;
}

int check_sight(const ttmi_paged_sight* sight) {
  TTMI_REQUIRE(sight != nullptr, "sight is null");
  TTMI_REQUIRE(sight->window >= 0 && sight->sinks >= 0 && sight->family_count >= 0 && sight->max_shared >= 0,
               "window, sinks, family_count and max_shared must not be negative");
  TTMI_REQUIRE((reinterpret_cast<uintptr_t>(sight->families) & 3) == 0, "families is not aligned to its elements");
  return 0;
}

// What both forms of the call check; the arguments that they have in common.
int attention_args(const void* q, int64_t q_pitch, void* out, int64_t out_pitch, int64_t heads, const ttmi_paged_cache* cache, const ttmi_paged_batch* batch,
                   int64_t max_tokens, int64_t max_length, float scale, int causal, int64_t window, int dtype, PagedArgs* a) {
  if (int rc = paged_view(cache, batch, heads, &a->view)) return rc;
  const int64_t d = cache->head_dim;
  TTMI_REQUIRE(d == 64 || d == 128, "paged attention needs head_dim 64 or 128");
  TTMI_REQUIRE(q_pitch >= heads * d && out_pitch >= heads * d, "rows overlap: a pitch is too small");
  TTMI_REQUIRE(dtype == TTMI_F32 || dtype == TTMI_F16 || dtype == TTMI_BF16, "unsupported dtype");
  TTMI_REQUIRE(window >= 0 && max_tokens >= 0 && max_length >= 0, "window, max_tokens and max_length must not be negative");
  // (a launch has less than 2^32 threads: 512 of them for a sequence and key/value head, or 256 for 128 rows besides)
  TTMI_REQUIRE(batch->tokens * heads < 1 << 30 && batch->batch * cache->kv_heads < 1 << 23, "more rows or sequences than one launch takes");
  a->scale_log2e = scale * 1.4426950408889634f;
  TTMI_REQUIRE(scale > 0.f && a->scale_log2e <= std::numeric_limits<float>::max(), "scale must be positive, and finite times log2(e)");
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  TTMI_REQUIRE(q != nullptr && out != nullptr, "q or out is null");
  TTMI_REQUIRE(rows_aligned(q, q_pitch, dtype) && rows_aligned(out, out_pitch, dtype), "rows of q and out must be 16-byte aligned");
  a->q = q, a->out = out, a->keys = cache->keys, a->values = cache->values, a->q_pitch = q_pitch, a->out_pitch = out_pitch;
  a->heads = (int)heads, a->group = (int)(heads / cache->kv_heads), a->causal = causal != 0;
  a->window = (int)std::min(window, kWidest);
  a->sinks = 0, a->families = nullptr;
  return 0;
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
  if (int rc = attention_args(q, q_pitch, out, out_pitch, heads, cache, batch, max_tokens, max_length, scale, causal, window, dtype, &a)) return rc;
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  const int64_t d = cache->head_dim;
  const PagedPlan p = plan(a.view, heads, max_tokens, max_length, window, dtype);
  const int64_t bytes = (p.few_floats + p.tile_floats) * 4;
  TTMI_REQUIRE(bytes == 0 || (workspace != nullptr && workspace_bytes >= bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "the workspace is too small or not 16-byte aligned");
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

int ttmi_paged_attention_sight_workspace(const ttmi_paged_cache* cache, const ttmi_paged_batch* batch, int64_t heads, int64_t max_tokens, int64_t max_length,
                                         const ttmi_paged_sight* sight, int dtype, int64_t* bytes) {
  if (int rc = check_sight(sight)) return rc;
  PagedView view;
  TTMI_REQUIRE(bytes != nullptr, "bytes is null");
  if (int rc = paged_view(cache, batch, heads, &view)) return rc;
  ttmi_paged_sight used = *sight;
  if (!sharing_pays(view, heads, max_tokens, max_length, used, dtype)) used.families = nullptr;
  if (used.families == nullptr && (used.sinks == 0 || used.window == 0))
    return ttmi_paged_attention_workspace(cache, batch, heads, max_tokens, max_length, used.window, dtype, bytes);
  TTMI_REQUIRE(max_tokens >= 0 && max_length >= 0, "max_tokens and max_length must not be negative");
  *bytes = batch->tokens == 0 || batch->batch == 0 ? 0 : plan_sight(view, heads, max_tokens, max_length, used, dtype).floats * 4;
  return 0;
}

int ttmi_paged_attention_sight(const void* q, int64_t q_pitch, void* out, int64_t out_pitch, int64_t heads, const ttmi_paged_cache* cache,
                               const ttmi_paged_batch* batch, int64_t max_tokens, int64_t max_length, float scale, int causal, const ttmi_paged_sight* sight,
                               void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  if (int rc = check_sight(sight)) return rc;
  SightLaunch l;
  PagedArgs& a = l.all;
  if (int rc = attention_args(q, q_pitch, out, out_pitch, heads, cache, batch, max_tokens, max_length, scale, causal, sight->window, dtype, &a)) return rc;
  if (batch->tokens == 0 || batch->batch == 0) return 0;
  ttmi_paged_sight used = *sight;
  if (!sharing_pays(a.view, heads, max_tokens, max_length, used, dtype)) used.families = nullptr;
  if (used.families == nullptr && (used.sinks == 0 || used.window == 0))
    return ttmi_paged_attention(q, q_pitch, out, out_pitch, heads, cache, batch, max_tokens, max_length, scale, causal, used.window, workspace, workspace_bytes,
                                dtype, stream);
  const SightPlan p = plan_sight(a.view, heads, max_tokens, max_length, used, dtype);
  const int64_t kv_heads = cache->kv_heads, tile_groups = p.own_blocks * kv_heads * p.own.tile_splits, few_groups = p.own.few_splits > 0 ? p.own.few_splits : batch->batch * kv_heads;
  TTMI_REQUIRE(p.shares + tile_groups + (p.own.few ? few_groups : 0) < 1 << 24, "more rows or sequences than one launch takes");
  TTMI_REQUIRE(p.floats == 0 || (workspace != nullptr && workspace_bytes >= p.floats * 4 && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "the workspace is too small or not 16-byte aligned");
  a.sinks = (int)std::min(used.sinks, kWidest), a.families = used.families;
  a.partial = static_cast<float*>(workspace);
  a.every = !p.own.few, a.chunk = p.own.tile_chunk, a.splits = p.own.tile_splits, a.ordered = 1;
  a.shares = p.shares, a.family_splits = p.family_splits, a.family_least = p.family_least, a.family_few = p.family_few;
  a.own_at = p.few_rows, a.family_at = a.own_at + p.own_rows, a.whole_at = a.family_at + p.family_rows, a.rows = a.whole_at + p.whole_rows;
  l.run_tiles = p.own.tiles || p.shares > 0;
  a.run_few = p.own.few, a.few = p.own.few_rows, a.few_splits = p.own.few_splits, a.few_every = !p.own.tiles;
  a.own_blocks = p.own_blocks, a.tile_groups = (int)tile_groups;
  l.few = a;
  l.few.splits = p.own.few_splits;
  l.few.waves = l.run_tiles && a.view.page_shift >= 4 ? 4 : p.own.few_waves;  // (4 in one launch with the others)
  const auto launch = dtype == TTMI_F32 ? launch_sight_f32 : dtype == TTMI_F16 ? launch_sight_f16 : launch_sight_bf16;
  launch(l, cache->head_dim, static_cast<hipStream_t>(stream));
  return launch_status("paged_attention_sight");
}

}  // extern "C"
