"""Norms of heads in the append, attention with windows and first tokens that stay visible, and families of sequences that share their first pages, against the
formulas in 64 bits."""
import ctypes
import math
import random

import numpy as np
import pytest
import torch

import turbotransformers_amd as tt
from helpers import TORCH_DTYPES
from test_paged_gpu import DTYPES, E32, EPS, Case, turned
from turbotransformers_amd import capi

pytestmark = pytest.mark.gpu


class Sight(Case):
    """A batch with families.  families: (sequences, keys they have in common) in order; the common keys' full pages are the first one's, and what would have been the
    others' pages holds NaN."""

    def __init__(self, dt, new, past, heads, kv_heads, d, page, families=(), **kw):
        super().__init__(dt, new, past, heads, kv_heads, d, page, **kw)
        self.rows = np.array([[b, b + 1, 0] for b in range(len(new))], np.int32).reshape(-1, 3)
        first = 0
        for members, keys in families:
            self.share(first, first + members, keys)
            first += members
        self.families = any(row[2] for row in self.rows)

    def share(self, first, end, keys):
        n = keys // self.page
        for b in range(first + 1, end):
            own = self.table[b, :n].tolist()
            self.keys[own], self.values[own] = math.nan, math.nan
            self.table[b, :n] = self.table[first, :n]
        self.rows[first:end] = (first, end, n * self.page)

    def attention(self, causal=True, window=0, sinks=0, scale=None):
        """-> (out, tolerance), as Case.attention, whose docstring derives the tolerance (joining partial results of a family's keys and of a sequence's own is one
        join, as that of parts is)."""
        scale = scale if scale is not None else 1 / math.sqrt(self.d)
        eps = EPS[self.dt]
        out = torch.full((self.tokens, self.heads, self.d), math.nan, dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        for b, n in enumerate(self.lengths):
            rows = slice(int(self.starts[b]), int(self.starts[b + 1]))
            m = rows.stop - rows.start
            if m == 0:
                continue
            k, v = self.history(b, self.keys), self.history(b, self.values)
            position, key = torch.arange(n - m, n)[:, None], torch.arange(n)[None]
            hidden = key > position if causal else torch.zeros(m, n, dtype=torch.bool)
            if window:
                hidden = hidden | ((key <= position - window) & (key >= sinks))
            for h in range(self.heads):
                q = self.q[rows, h].double()
                kh, vh = k[:, h // group], v[:, h // group]
                s = (q @ kh.T * scale).masked_fill(hidden, -math.inf)
                size = (q.abs() @ kh.abs().T * scale).masked_fill(hidden, 0)
                top = s.amax(1, keepdim=True) if n else torch.zeros(m, 1)
                p = torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top)).masked_fill(hidden, 0)
                total = p.sum(1, keepdim=True)
                p = torch.where(total > 0, p / total, torch.zeros_like(p))
                o, a = p @ vh, p @ vh.abs()
                ds = (self.d + 6) * E32 * (size.amax(1, keepdim=True) if n else 0)
                t = a * (4 * ds + 2 * (n + 8) * E32 + 8 * E32) + eps / 2 * o.abs()
                if self.dt != "f32":
                    t = t + eps * a
                if self.dt == "f16" and n:
                    t = t + 2 * n * 2.0 ** -25 * vh.abs().max()
                out[rows, h], tol[rows, h] = o, t
        return out, tol

    def run_attention(self, families=None, hints=(0, 0), **kw):
        """hints: family_count and max_shared.  Where neither is known families are made use of however little there is to gain; None: both as they are."""
        rows = self.rows if families is None else np.asarray(families, np.int32)
        if self.families or families is not None:
            count, most = (len({row[0] for row in rows.tolist() if row[2]}), int(rows[:, 2].max())) if hints is None else hints
            kw.update(families=torch.from_numpy(rows.copy()).cuda(), family_count=count, max_shared=most)
        return super().run_attention(**kw)


def check(*args, causal=True, window=0, sinks=0, scale=None, **kw):
    case = Sight(*args, **kw)
    got = case.run_attention(causal=causal, window=window, sinks=sinks, scale=scale)
    want = case.check_attention(got, causal=causal, window=window, sinks=sinks, scale=scale)
    if case.families:
        _, tol = case.attention(causal=causal, window=window, sinks=sinks, scale=scale)
        n = int(case.starts[-1])
        hinted = case.run_attention(causal=causal, window=window, sinks=sinks, scale=scale, hints=None).cpu().double()
        assert ((hinted[:n] - want[:n]).abs() <= tol[:n]).all()
    assert (got[int(case.starts[-1]):] == 7.0).all()  # rows behind the last sequence are left as they were


# ------------------------------------------------------------------------------------------- windows and first tokens ------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (50, 31), (64, 64), (100, 33), (33, 200), (10000, 4), (5, 10000)])
def test_windows_with_sinks(dt, d, window, sinks):
    """Single tokens, chunks, prompts that begin before the window does, sequences without new tokens; first keys that end anywhere in a tile or reach into the window."""
    check(dt, [1, 90, 1, 0, 7, 40], [300, 40, 0, 50, 129, 0], 4, 2, d, 16, window=window, sinks=sinks, spare_rows=2, spare_width=1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,page", [(2, 2, 1), (6, 2, 2), (8, 1, 8), (32, 2, 32), (20, 1, 128), (4, 4, 4096)])
def test_windows_with_sinks_heads_and_pages(dt, heads, kv_heads, page):
    check(dt, [1, 20, 1, 3], [700, 400, 5, 260], heads, kv_heads, 64, page, window=70, sinks=9)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 3), (40, 17), (128, 128)])
def test_windows_with_sinks_without_causality(dt, window, sinks):
    check(dt, [1, 70, 3, 20], [5, 30, 400, 900], 4, 2, 64, 16, causal=False, window=window, sinks=sinks)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_long_windows_with_sinks_are_cut_and_joined(dt, causal):
    for window, sinks, new, past in ((1000, 4, [40], [5000]), (700, 300, [130, 9, 20], [2999, 100, 4000]), (2000, 70, [20], [1500]), (3000, 5, [1, 2], [9000, 3500]),
                                     (20, 3000, [30, 1], [5000, 6000])):
        check(dt, new, past, 4, 2, 64, 16, causal=causal, window=window, sinks=sinks, spare_rows=1)
    case = Sight(dt, [90, 30, 1], [3000, 17, 4000], 4, 2, 64, 16)
    for most in ((30, 400), (0, 0), (1 << 30, 1 << 40)):
        got = case.run_attention(max_tokens=most[0], max_length=most[1], window=900, sinks=77, causal=causal)
        case.check_attention(got, window=900, sinks=77, causal=causal)


@pytest.mark.parametrize("dt", DTYPES)
def test_sinks_without_a_window_say_nothing(dt):
    case = Sight(dt, [1, 40], [600, 100], 4, 2, 64, 16)
    assert torch.equal(case.run_attention(sinks=5), case.run_attention())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new,past", [([1, 5, 150], [300, 290, 200]), ([1], [9000]), ([60], [5000]), ([1] * 70, [400 + i for i in range(70)])])
def test_what_is_not_finite_reaches_only_the_tokens_that_see_it(dt, bad, new, past):
    """A value among the first keys that are seen, one behind them, one at the window's edge: other rows and columns keep their bits."""
    window, sinks = 100, 5
    case = Sight(dt, new, past, 4, 2, 64, 16)
    clean = case.run_attention(window=window, sinks=sinks).cpu()
    case.check_attention(clean, window=window, sinks=sinks)
    kept = case.values.clone()
    for key in (lambda n, p: 4, lambda n, p: 5, lambda n, p: 31, lambda n, p: p - window, lambda n, p: p - window + 1, lambda n, p: p + n - 1):
        case.values.copy_(kept)
        spoiled = torch.zeros(case.q.shape, dtype=torch.bool)
        for b, (n, p) in enumerate(zip(new, past)):
            at = key(n, p)
            case.values[case.table[b, at // 16], 1, at % 16, 7] = bad
            for i in range(n):
                spoiled[int(case.starts[b]) + i, 2:, 7] = at <= p + i and (at > p + i - window or at < sinks)
        got = case.run_attention(window=window, sinks=sinks).cpu()
        assert torch.equal(~torch.isfinite(got), spoiled)
        assert torch.equal(got[~spoiled], clean[~spoiled])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", ["keys", "queries"])
def test_numbers_near_the_largest(d, what):
    """fp32 products are taken apart into those of narrower numbers, which the largest ones are not: scores of moderate size from a factor beyond 2^127 and one that makes up for it."""
    case = Sight("f32", [140, 30, 3], [0, 90, 300], 4, 2, d, 16)
    case.check_attention(case.run_attention(window=50, sinks=7), window=50, sinks=7)
    small = 2.0 ** -125 * (1 + torch.rand(case.q.shape[:2], generator=torch.Generator().manual_seed(3)))  # (2^127.99 times 2^-124 at most, times the scale)
    if what == "keys":
        case.q[..., 5] = small
        for b, position in ((0, 2), (0, 77), (0, 130), (1, 100), (2, 301)):
            case.keys[case.table[b, position // 16], :, position % 16, 5] = 3.4e38 if position % 2 else -2.0 ** 127
    else:
        case.keys[..., 5] = torch.where(torch.isnan(case.keys[..., 5]), case.keys[..., 5], torch.full_like(case.keys[..., 5], 2.0 ** -125))
        for row in (0, 31, 64, 139, 150, 171):
            case.q[row, 1, 5], case.q[row, 2, 5] = 3.4028234e38, -1.9e38
    case.check_attention(case.run_attention(window=50, sinks=7), window=50, sinks=7)


@pytest.mark.parametrize("d", [64, 128])
def test_keys_near_the_largest_in_common(d):
    case = Sight("f32", [40, 30, 20, 1, 1], [300, 256, 270, 400, 300], 4, 2, d, 16, families=[(3, 256), (2, 288)])
    case.q[..., 5] = 2.0 ** -125
    for b, position in ((0, 2), (0, 77), (0, 255), (1, 280), (3, 5), (3, 288)):
        case.keys[case.table[b, position // 16], :, position % 16, 5] = 3.4e38 if position % 2 else -2.0 ** 127
    case.check_attention(case.run_attention())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [3.4e38, math.inf, 0.0])
def test_what_lies_behind_the_last_key_and_under_the_gap(d, bad):
    """Slots that no token sees may hold anything (NaN otherwise, here); the bits are the same."""
    case = Sight("f32", [140, 30, 2], [400, 90, 37], 4, 2, d, 16)
    outs = []
    for fill in (math.nan, bad):
        case.keys, case.values = (torch.where(torch.isnan(x), torch.full_like(x, fill), x) for x in (case.keys, case.values))
        case.keys[case.table[0, 10:20]], case.values[case.table[0, 10:20]] = fill, fill  # (positions 160 to 319; the first new token's window begins at 351)
        outs.append(case.run_attention(window=50, sinks=7).cpu()[:172])
    assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", ["keys", "queries", "values", "a column of keys", "a column of queries", "one value of each sequence", "scale"])
@pytest.mark.parametrize("e", [97, 101, 112, 120, 125])
def test_numbers_far_from_one(d, what, e):
    """Numbers whose parts would fall below those that bf16 has, with factors that make up for it: the tolerance of fp32 as ever, in the kernels with and without first tokens, chunks,
    families and single tokens.  (Results below the normal numbers: each product and each of their sums is off by up to 2^-150 besides, against a sum of probabilities of at least 1, and
    so is the result.)"""
    new, past = [140, 30, 3, 1], [0, 90, 300, 200]
    for families, window, sinks in (((), 50, 7), ((), 50, 0), (((2, 0), (2, 192)), 0, 0), (((2, 0), (2, 192)), 60, 5)):
        case = Sight("f32", new, past, 4, 2, d, 16, families=families)
        scale = 1 / math.sqrt(d)
        if what == "keys":
            case.keys, case.q = case.keys * 2.0 ** -e, case.q * 2.0 ** e
        elif what == "queries":
            case.q, case.keys = case.q * 2.0 ** -e, case.keys * 2.0 ** e
        elif what == "values":
            case.values = case.values * 2.0 ** -e
        elif what == "a column of keys":
            case.keys[..., 5], case.q[..., 5] = case.keys[..., 5] * 2.0 ** -e, case.q[..., 5] * 2.0 ** e
        elif what == "a column of queries":
            case.q[..., 5], case.keys[..., 5] = case.q[..., 5] * 2.0 ** -e, case.keys[..., 5] * 2.0 ** e
        elif what == "one value of each sequence":  # that stands alone in its column
            case.values[..., 7] = torch.where(torch.isnan(case.values[..., 7]), case.values[..., 7], torch.zeros_like(case.values[..., 7]))
            for b, n in enumerate(case.lengths):
                case.values[case.table[b, (n - 2) // 16], :, (n - 2) % 16, 7] = 1.2345678 * 2.0 ** -e
        else:
            case.q, case.keys, scale = case.q * 2.0 ** -(e // 2), case.keys * 2.0 ** -(e // 2), scale * 2.0 ** (2 * (e // 2))
        got = case.run_attention(window=window, sinks=sinks, scale=scale).cpu().double()
        want, tol = case.attention(window=window, sinks=sinks, scale=scale)
        assert ((got - want).abs() <= tol + (2 * max(case.lengths) + 1) * 2.0 ** -150).all(), (families, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,past,window,sinks,families", [([140, 30, 2], [400, 90, 37], 50, 7, ()), ([40], [5000], 1000, 7, ()), ([150], [0], 1000, 20, ()), ([20, 30, 1], [300, 290, 270], 0, 0, ((3, 256),)),
                                                            ([20, 30, 1], [1300, 1290, 1270], 100, 9, ((3, 1256),))])
def test_small_numbers_that_no_token_sees(d, new, past, window, sinks, families):
    """Behind a sequence's last key and in the gap of its window they change no bit, as others do not."""
    case = Sight("f32", new, past, 4, 2, d, 16, families=families)
    outs = []
    for fill in (math.nan, 2.0 ** -120):
        case.keys, case.values = (torch.where(torch.isnan(x), torch.full_like(x, fill), x) for x in (case.keys, case.values))
        for b, p in enumerate(past):  # (whole pages that lie under the gap of the first new token and so of all: in a family, of its sequence with the fewest)
            p = min(past) if families else p
            if window and p - window > sinks:
                pages = case.table[b, -(-sinks // 16):(p + 1 - window) // 16]
                case.keys[pages], case.values[pages] = fill, fill
        outs.append(case.run_attention(window=window, sinks=sinks).cpu()[:sum(new)])
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])
    case.keys, case.values = torch.zeros_like(case.keys), torch.zeros_like(case.values)
    assert (case.run_attention(window=window, sinks=sinks)[:sum(new)] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_minus_infinity(d):
    """A key with a score of minus infinity weighs nothing, whether it comes from an infinity or from numbers near it: the bits are those of a score that is merely low."""
    case = Sight("f32", [140, 30], [0, 90], 4, 2, d, 16)
    case.q[..., 5] = -1.0
    outs = []
    for low in (3000.0, 3.4e38, math.inf):
        for b, position in ((0, 2), (0, 77), (1, 100)):
            case.keys[case.table[b, position // 16], :, position % 16, 5] = low
        outs.append(case.run_attention(window=50, sinks=7).cpu())
    assert torch.isfinite(outs[0]).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ------------------------------------------------------------------------------------------------------- families ------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (16, 1)])
def test_families_of_single_tokens(dt, d, heads, kv_heads):
    """Two and more samples of texts that end around the steps of sharing, some alone, some with nothing of their own but the new token."""
    families = [(3, 128), (1, 0), (2, 127), (5, 144), (4, 256), (1, 0), (2, 640), (3, 16), (2, 0)]
    rng = random.Random(heads)
    past = [keys + rng.choice([0, 1, 15, 16, 60, 200]) for members, keys in families for _ in range(members)]
    check(dt, [1] * len(past), past, heads, kv_heads, d, 16, families=families, spare_rows=3, spare_width=1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("members,keys,heads,kv_heads", [(2, 3000, 4, 4), (40, 1500, 8, 2), (9, 5000, 16, 1), (70, 700, 4, 2), (3, 9000, 6, 2)])
def test_long_families_are_cut_and_joined(dt, members, keys, heads, kv_heads):
    rng = random.Random(members)
    past = [keys + rng.choice([1, 30, 200, 900 if i % 9 == 0 else 40]) for i in range(members)]
    check(dt, [1] * members, past, heads, kv_heads, 64, 16, families=[(members, keys)])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (200, 1, 64)])
def test_families_with_chunks(dt, heads, kv_heads, d):
    """Questions of many tokens about a text, speculated tokens, sequences without new tokens, the first of a family among them."""
    check(dt, [20, 1, 0, 130, 3, 0, 5, 1, 1, 16], [700, 650, 900, 640, 645, 512, 520, 513, 90, 40], heads, kv_heads, d, 16,
          families=[(5, 640), (3, 512), (2, 0)], spare_rows=1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page", [1, 2, 8, 16, 128, 256])
def test_families_and_page_sizes(dt, page):
    check(dt, [1, 2, 1, 1, 40], [600, 530, 700, 300, 512], 4, 2, 64, page, families=[(3, 512), (2, 256)])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_new_tokens_among_the_common_keys(dt, causal):
    """A family's keys are the first of its sequences, whatever is new: tokens that see a part of them, one of them, none."""
    case = Sight(dt, [300, 1, 200, 40, 1], [0, 299, 100, 260, 600], 4, 2, 64, 16, families=[(4, 256), (1, 0)])
    case.check_attention(case.run_attention(causal=causal), causal=causal)
    case = Sight(dt, [1, 1, 20], [400, 500, 380], 4, 2, 64, 16, families=[(3, 384)])
    case.lengths[2] = 7  # its 20 tokens have positions -13 to 6
    got = case.run_attention(max_length=501)
    assert (got[2:15] == 0).all()
    case.check_attention(got)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 0), (700, 0), (100, 4), (300, 130), (50, 512), (200, 900), (10000, 7)])
def test_families_with_windows_and_sinks(dt, window, sinks):
    """Windows that end before the common keys, in them, and not at all; first keys that stay visible: some, the common ones, more."""
    check(dt, [1, 1, 30, 1, 1, 1, 0, 2], [900, 520, 600, 3000, 1, 700, 400, 2900], 4, 2, 64, 16, families=[(3, 512), (1, 0), (1, 0), (3, 384)], window=window,
          sinks=sinks, spare_rows=1)
    check(dt, [1] * 6, [2600, 2500, 2999, 2450, 5000, 2447], 8, 2, 128, 16, families=[(6, 2432)], window=window, sinks=sinks)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (1 << 40, 1 << 40), (7, 200), (1, 0), (0, 64), (1, 1 << 40)])
def test_hints_of_families_choose_nothing_but_the_cut(dt, hints):
    case = Sight(dt, [1, 40, 1, 1, 1, 3], [1600, 1400, 1500, 300, 260, 90], 8, 2, 64, 16, families=[(3, 1392), (2, 256), (1, 0)])
    case.check_attention(case.run_attention(hints=hints))
    case.check_attention(case.run_attention(hints=hints, max_tokens=1, max_length=10))


def test_rows_of_families_that_disagree_are_sequences_on_their_own():
    """Numbers outside the batch, firsts that name another first or an end before the sequence, families that claim each other's sequences: no key is lost or read twice."""
    case = Sight("f16", [1, 2, 1, 1, 30, 1], [700, 600, 650, 620, 610, 640], 8, 2, 64, 16, families=[(6, 512)])
    big = 1 << 31
    for rows in ([[0, 6, 0]] * 6, [[0, 6, -5]] * 6, [[-1, 6, 512]] * 6, [[9, 6, 512]] * 6, [[big - 1, big - 1, big - 1]] * 6, [[-big, -big, -big]] * 6, [[0, 3, 512]] * 6,
                 [[0, 6, 512]] * 3 + [[3, 6, 256]] * 3, [[1, 6, 512], [0, 6, 512]] + [[0, 6, 512]] * 4, [[0, 6, 512], [0, 2, 256], [2, 6, 512], [2, 6, 512], [0, 6, 512], [4, 9, 400]],
                 [[5, 6, 512]] * 5 + [[5, 6, 512]], [[0, 6, 512]] + [[b, b + 1, 512] for b in range(1, 6)], [[0, 0, 512]] * 6):
        case.check_attention(case.run_attention(families=rows))
    # more keys promised than lie in the same pages: they are read from the first sequence's, whose own result that is
    got = case.run_attention(families=[[0, 100, big - 1]] * 6)
    want, tol = case.attention()
    assert ((got[0].cpu().double() - want[0]).abs() <= tol[0]).all()
    tt.cxx.synchronize()


class Apart(Sight):
    """A family of the sequences `first` to `end`, all behind the same `keys` tokens but for those of `others`, {sequence: (its row, tokens that it has in common)}.  What
    would have been the pages of common tokens holds NaN."""

    def __init__(self, dt, new, past, heads, kv_heads, d, page, first, end, keys, others, **kw):
        super().__init__(dt, new, past, heads, kv_heads, d, page, **kw)
        for b in range(first, end):
            row, common = others.get(b, ((first, end, keys), keys))
            n = common // page if b > first else 0
            own = self.table[b, :n].tolist()
            self.keys[own], self.values[own] = math.nan, math.nan
            self.table[b, :n] = self.table[first, :n]
            self.rows[b] = row
        self.families = True


ROWS_THAT_DIFFER = [((0, 6, 0), 0), ((0, 6, 128), 128), ((0, 6, 128), 0), ((0, 6, 256), 128), ((0, 6, 511), 0), ((0, 6, 640), 0), ((0, 6, -512), 0), ((0, 5, 512), 0),
                    ((0, 7, 512), 256), ((0, 2, 512), 0), ((0, 1 << 30, 512), 0), ((1, 6, 512), 0)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new", [[1] * 6, [1, 20, 130, 1, 1, 5]])
@pytest.mark.parametrize("heads,page", [(4, 16), (8, 16), (8, 4)])
def test_a_sequence_whose_row_differs_from_the_firsts_reads_its_own_pages(dt, new, heads, page):
    """Sequences that name the first of a family and say another end or another number of keys, none among them, hold other pages: each its own tokens' attention, in the
    kernels for few and for many rows, in the middle of a family's rows and at their end."""
    for row, common in ROWS_THAT_DIFFER:
        for window, sinks in ((0, 0), (300, 140)):
            case = Apart(dt, new, [600, 530, 700, 512, 650, 590], heads, 2, 64, page, 0, 6, 512, {2: (row, common), 5: (row, common)})
            case.check_attention(case.run_attention(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("batch", [80, 300])
@pytest.mark.parametrize("chunks", [False, True])
def test_rows_that_differ_across_the_bounds_of_64_sequences(dt, batch, chunks):
    """A family whose first sequence is among other 64 than some that name it, with and without a row like its."""
    first, end = batch - 25, batch
    others = {b: ((first, end, says), 0) for b, says in ((first + 2, 0), (first + 3, 256), (end - 6, 0), (end - 5, 256), (end - 1, 0))}
    new = [3 if chunks and b % 5 == 0 else 1 for b in range(batch)]
    case = Apart(dt, new, [3] * first + [130 + b % 3 for b in range(25)], 32, 2, 64, 16, first, end, 128, others)
    case.check_attention(case.run_attention())
    case = Apart(dt, new, [3] * 60 + [130 + b % 3 for b in range(20)] + [3] * (batch - 80), 32, 2, 64, 16, 60, 80, 128,
                 {b: ((60, 80, says), 0) for b, says in ((62, 0), (65, 256), (70, 0), (79, 64))})
    case.check_attention(case.run_attention())


def test_a_sequence_leaves_its_family_between_replays():
    """A recorded step whose second sequence is switched off in the tensor of families, gets another text's pages, and comes back."""
    case = Sight("bf16", [1, 1, 1], [700, 690, 650], 8, 2, 64, 16, families=[(3, 640)])
    other = Case("bf16", [1], [690], 8, 2, 64, 16, seed=5)
    pages = case.keys.shape[0]
    keys, values = torch.cat((case.keys, other.keys)).nan_to_num().cuda(), torch.cat((case.values, other.values)).nan_to_num().cuda()
    table, starts, lengths = case.device_args()
    table.clamp_(0, pages - 1)
    rows = torch.from_numpy(case.rows).cuda()
    q = case.q.cuda()
    call = lambda: tt.paged_attention(q, keys, values, table, starts, lengths, max_tokens=1, max_length=701, families=rows)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    kept = table[1].clone()
    other.q = case.q[1:2]
    for away in (False, True, True, False):
        table[1] = kept
        rows[1, 2] = 0 if away else 640
        if away:
            table[1, :44] = torch.from_numpy(other.table[0, :44]).cuda() + pages
        graph.replay()
        torch.randn(1 << 16, device="cuda").sum()
        torch.cuda.synchronize()
        want, tol = case.attention()
        if away:
            want[1:2], tol[1:2] = other.attention()
        assert ((out.cpu().double() - want).abs() <= tol).all(), away
        out.fill_(math.nan)
    tt.cxx.synchronize()


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_common_keys_end_where_the_first_sequence_does(dt):
    """A row that promises more keys than the first sequence of the family has: what it has not is each sequence's own."""
    case = Sight(dt, [1, 1, 1], [300, 700, 650], 4, 2, 64, 16, families=[(3, 288)])
    case.check_attention(case.run_attention(families=[[0, 3, 640]] * 3))


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads", [(20, 4), (32, 8)])
def test_many_rows_of_many_heads_are_joined(dt, heads, kv_heads):
    """280 sequences, so many rows and heads that a wavefront joins several of them; families of 2 to 70, over the bounds of 64 sequences, some sequences with chunks."""
    rng = random.Random(7)
    families, left = [], 280
    while left:
        members = min(left, rng.choice([1, 2, 3, 9, 40, 70]))
        families.append((members, rng.choice([128, 144]) if members > 1 else 0))
        left -= members
    check(dt, [rng.choice([1, 1, 1, 1, 7]) for _ in range(280)], [rng.randint(144, 160) for _ in range(280)], heads, kv_heads, 64, 16, families=families)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("batch", [63, 64, 65, 200, 300])
def test_many_families(dt, batch):
    """More sequences than a wavefront has lanes, families across that border, some sequences without new tokens and some long ones."""
    rng = random.Random(batch)
    families, left = [], batch
    while left:
        members = min(left, rng.choice([1, 1, 2, 5, 17]))
        families.append((members, rng.choice([128, 200, 384]) if members > 1 else 0))
        left -= members
    past = [keys + rng.choice([0, 3, 70, 1500 if rng.random() < 0.1 else 130]) for members, keys in families for _ in range(members)]
    new = [0 if i % 7 == 3 else 1 for i in range(batch)]
    check(dt, new, past, 4, 2, 64, 16, families=families, spare_rows=1)
    new = [40 if i % 31 == 0 else m for i, m in enumerate(new)]
    check(dt, new, past, 4, 2, 64, 16, families=families)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("pairs,page", [(40, 16), (330, 16), (40, 4)])
def test_more_parts_of_families_than_workgroups(dt, pairs, page):
    """Families of two sequences with up to 72 rows a key/value head, of other lengths each, said to be one short family: workgroups take several of their parts."""
    rng = random.Random(pairs)
    families = [(2, rng.choice([128, 130, 300])) for _ in range(pairs)]
    past = [keys + rng.choice([0, 5]) for members, keys in families for _ in range(members)]
    case = Sight(dt, [1] * len(past), past, 72, 2, 64, page, families=families)
    want, tol = case.attention()
    for hints in ((0, 0), (0, 64)):
        got = case.run_attention(hints=hints).cpu().double()
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new,past", [([1, 1, 1], [700, 650, 600]), ([30, 1, 20], [700, 650, 600])])
def test_queries_that_are_not_finite_spoil_their_own_row(dt, new, past):
    case = Sight(dt, new, past, 8, 2, 64, 16, families=[(3, 592)])
    clean = case.run_attention().cpu()
    case.check_attention(clean)
    spoiled = torch.zeros(clean.shape, dtype=torch.bool)
    for b, head in ((0, 1), (2, 5)):
        case.q[int(case.starts[b]), head, 3] = math.nan
        spoiled[int(case.starts[b]), head] = True
    got = case.run_attention().cpu()
    assert torch.equal(torch.isnan(got), spoiled) and torch.equal(got[~spoiled], clean[~spoiled])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new,past", [([1, 30, 1, 1], [700, 300, 400, 500]), ([1, 3, 1, 1], [700, 316, 400, 500])])
def test_what_is_not_finite_in_common_keys(dt, bad, new, past):
    """A value of a common key reaches every token that sees it, in its column alone; one behind every token's position, or in front of some tokens' windows, only those who see it."""
    window = 330
    case = Sight(dt, new, past, 4, 2, 64, 16, families=[(4, 320)])  # (tokens 300 to 319 of the second sequence are common keys)
    for w in (0, window):
        clean = case.run_attention(window=w).cpu()
        case.check_attention(clean, window=w)
        kept = case.values.clone()
        for key in (0, 63, 100, 255, 310, 319):
            case.values[case.table[0, key // 16], 1, key % 16, 7] = bad
            spoiled = torch.zeros(case.q.shape, dtype=torch.bool)
            for b, (n, p) in enumerate(zip(new, past)):
                for i in range(n):
                    spoiled[int(case.starts[b]) + i, 2:, 7] = key <= p + i and (w == 0 or key > p + i - w)
            got = case.run_attention(window=w).cpu()
            assert torch.equal(~torch.isfinite(got), spoiled), (w, key)
            assert torch.equal(got[~spoiled], clean[~spoiled]), (w, key)
            case.values.copy_(kept)
    case.q[:, 0, 0] = -math.inf  # scores of minus infinity alone: NaN; among others: weights of zero
    case.keys[..., 0] = torch.where(torch.isnan(case.keys[..., 0]), case.keys[..., 0], torch.ones_like(case.keys[..., 0]))
    got = case.run_attention().cpu()
    assert torch.isnan(got[:, 0]).all() and torch.isfinite(got[:, 1:]).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_scores_far_apart_in_common_and_own_keys(dt):
    case = Sight(dt, [1, 30, 1], [900, 800, 790], 4, 2, 64, 16, families=[(3, 768)], scale_q=30.0)
    case.check_attention(case.run_attention())
    for scale in (1e-4, 3.0):
        case.check_attention(case.run_attention(scale=scale), scale=scale)


def test_the_same_call_twice_gives_the_same_bits():
    for dt in DTYPES:
        case = Sight(dt, [1, 40, 1, 1, 1], [3000, 2000, 2700, 300, 20], 8, 2, 128, 16, families=[(3, 1984), (2, 0)])
        assert torch.equal(case.run_attention(), case.run_attention())
        assert torch.equal(case.run_attention(window=700, sinks=40), case.run_attention(window=700, sinks=40))


@pytest.mark.parametrize("dt", DTYPES)
def test_offsets_beyond_32_bits(dt):
    """A cache of more than 2^32 bytes whose last pages hold the common and the own keys."""
    d, page, kv_heads = 128, 64, 8
    pages = (1 << 31) // (kv_heads * page * d) + 60
    keys = torch.zeros((pages, kv_heads, page, d), dtype=TORCH_DTYPES[dt], device="cuda")
    values = torch.zeros_like(keys)
    case = Sight(dt, [1, 20, 1], [500, 437, 440], 16, kv_heads, d, page, families=[(3, 384)])
    used = sorted({int(p) for row, n in zip(case.table, case.lengths) for p in row[:-(-n // page)]})
    high = {p: pages - 1 - i for i, p in enumerate(used)}
    for p, h in high.items():
        keys[h], values[h] = case.keys[p].cuda(), case.values[p].cuda()
    table = torch.tensor([[high.get(int(p), 0) for p in row] for row in case.table], dtype=torch.int32, device="cuda")
    _, starts, lengths = case.device_args()
    rows = torch.from_numpy(case.rows).cuda()
    for window, sinks in ((0, 0), (60, 30)):
        got = tt.paged_attention(case.q.cuda(), keys, values, table, starts, lengths, max_length=600, families=rows, window=window, sinks=sinks)
        case.check_attention(got, window=window, sinks=sinks)
    norm = torch.ones(d, device="cuda")
    qkv = torch.randn(case.tokens, 32, d, device="cuda").to(keys.dtype)
    tt.rotary_append(qkv, keys, values, table, starts, lengths, q_norm=norm, k_norm=norm)
    last = int(table[1, (case.lengths[1] - 1) // page])
    assert torch.equal(values[last, :, (case.lengths[1] - 1) % page], qkv[20, 24:])
    tt.cxx.synchronize()


@pytest.mark.parametrize("new", [[1, 30, 1, 1], [1, 1, 1, 1]])
def test_pages_outside_the_cache_are_reported(new):
    case = Sight("f16", new, [400, 307, 290, 100], 4, 2, 64, 16, families=[(3, 256), (1, 0)])
    case.keys, case.values = case.keys.nan_to_num(), case.values.nan_to_num()
    for kw in (dict(families=torch.from_numpy(case.rows).cuda()), dict(window=200, sinks=20), dict(families=torch.from_numpy(case.rows).cuda(), window=200, sinks=20)):
        for bad in (-1, 1 << 20):
            for column in (1, 17):
                table, starts, lengths = case.device_args()
                table[0, column] = bad
                out = tt.paged_attention(case.q.cuda(), case.keys.cuda(), case.values.cuda(), table, starts, lengths, **kw)
                torch.cuda.synchronize()
                with pytest.raises(tt.cxx.EnforceNotMet, match="out of range"):
                    tt.cxx.synchronize()
                tt.cxx.synchronize()  # reported once
                want, tol = case.attention(window=kw.get("window", 0), sinks=kw.get("sinks", 0))
                assert ((out.cpu().double() - want).abs() <= tol)[-1].all()  # the sequence that is on its own
    # more keys than the table has pages for: those there are
    table, starts, lengths = case.device_args()
    lengths[0] = 5000
    tt.paged_attention(case.q.cuda(), case.keys.cuda(), case.values.cuda(), table.clamp(0, 3)[:, :20].contiguous(), starts, lengths, window=100, sinks=3)
    torch.cuda.synchronize()
    with pytest.raises(tt.cxx.EnforceNotMet, match="out of range"):
        tt.cxx.synchronize()


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_that_lie_apart(dt):
    case = Sight(dt, [1, 20, 1], [300, 267, 290], 4, 2, 64, 16, families=[(3, 256)])
    wide = torch.zeros(case.tokens, 8 * 64, dtype=case.q.dtype, device="cuda")
    wide[:, 64:64 + 256] = case.q.cuda().view(-1, 256)
    result = torch.full((case.tokens, 512), 7.0, dtype=case.q.dtype, device="cuda")
    for kw in (dict(), dict(window=40, sinks=3)):
        got = tt.paged_attention(wide[:, 64:320], case.keys.cuda(), case.values.cuda(), *case.device_args(), out=result[:, 128:384],
                                 families=torch.from_numpy(case.rows).cuda(), **kw)
        case.check_attention(got, **kw)
        assert (result[:, :128] == 7).all() and (result[:, 384:] == 7).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_recorded_steps(dt):
    """A step recorded into two graphs and replayed with growing lengths, other tables and other families, eager work and synchronisations between the replays."""
    case = Sight(dt, [1, 1, 1, 1], [690, 600, 555, 30], 8, 2, 128, 16, families=[(3, 512), (1, 0)], spare_width=3)
    table, starts, lengths = case.device_args()
    table.clamp_(0, case.keys.shape[0] - 1)
    keys, values = case.keys.nan_to_num().cuda(), case.values.nan_to_num().cuda()
    qkv = torch.randn(4, 12, 128, generator=torch.Generator().manual_seed(2)).to(keys.dtype).cuda()
    inv_freq, norm, rows = tt.rotary_frequencies(128), torch.rand(128, device="cuda"), torch.from_numpy(case.rows).cuda()

    def call():
        q = tt.rotary_append(qkv, keys, values, table, starts, lengths, inv_freq, q_norm=norm, k_norm=norm)
        return (tt.paged_attention(q, keys, values, table, starts, lengths, max_tokens=1, max_length=720, families=rows),
                tt.paged_attention(q, keys, values, table, starts, lengths, max_tokens=1, max_length=720, window=300, sinks=70))

    call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for turn in range(4):
        qkv.copy_(torch.randn(4, 12, 128, generator=torch.Generator().manual_seed(10 + turn)).to(keys.dtype))
        lengths.add_(1)
        rows[:3, 2] = [512, 384, 0, 200][turn]
        want = call()
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            for x in out:
                x.fill_(math.nan)
            graph.replay()
            torch.randn(1 << 16, device="cuda").sum()
            torch.cuda.synchronize()
            assert all(torch.equal(x, w) for x, w in zip(out, want)), turn
    tt.cxx.synchronize()


def test_calls_on_two_streams_at_a_time():
    """Two batches with families in turn on two streams without waiting for one another: their workspaces are their own."""
    cases = [Sight("bf16", [1] * 3, [3000, 2000, 2900], 8, 2, 128, 16, seed=1, families=[(3, 1984)]),
             Sight("bf16", [40, 1], [2500, 1200], 8, 2, 128, 16, seed=2, families=[(2, 1200)])]
    tensors = [[x.cuda() for x in (case.q, case.keys, case.values)] + case.device_args() for case in cases]
    hints = [dict(max_tokens=max(case.new), max_length=max(case.lengths), families=torch.from_numpy(case.rows).cuda()) for case in cases]
    want = [tt.paged_attention(*t, **h) for t, h in zip(tensors, hints)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(tt.paged_attention(*tensors[i], **hints[i]))
    torch.cuda.synchronize()
    for i in range(2):
        cases[i].check_attention(want[i])
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_c_interface():
    """The calls through the C ABI: the workspace they ask for, and their refusal of a smaller one."""
    lib = capi.load()
    case = Sight("f16", [1, 1, 1], [5000, 4800, 20], 4, 1, 64, 16, families=[(2, 4800), (1, 0)])
    q, k, v = case.q.cuda(), case.keys.cuda(), case.values.cuda()
    table, starts, lengths = case.device_args()
    rows = torch.from_numpy(case.rows).cuda()
    cache = capi.PagedCache(k.data_ptr(), v.data_ptr(), k.shape[0], 1, 16, 64)
    batch = capi.PagedBatch(table.data_ptr(), table.shape[1], starts.data_ptr(), lengths.data_ptr(), 3, 3)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for window, sinks, families in ((0, 0, rows), (3000, 9, None), (3000, 9, rows), (0, 0, None), (0, 5, None)):
        sight = capi.PagedSight(window, sinks, families.data_ptr() if families is not None else None, 0, 0)
        n = ctypes.c_int64(-1)
        capi.check(lib.ttmi_paged_attention_sight_workspace(ctypes.byref(cache), ctypes.byref(batch), 4, 1, 5001, ctypes.byref(sight), capi.F16, ctypes.byref(n)))
        assert n.value >= 0
        work = torch.empty(max(16, n.value), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(q)
        call = lambda bytes: lib.ttmi_paged_attention_sight(q.data_ptr(), 256, out.data_ptr(), 256, 4, ctypes.byref(cache), ctypes.byref(batch), 1, 5001, 0.125, 1,
                                                            ctypes.byref(sight), work.data_ptr(), bytes, capi.F16, stream)
        capi.check(call(n.value))
        torch.cuda.synchronize()
        case.check_attention(out, window=window, sinks=sinks)
        if n.value:
            assert call(n.value - 1) == -1
    tt.cxx.synchronize()


def test_calls_without_tokens_or_sequences():
    case = Sight("f16", [1, 1], [300, 290], 4, 2, 64, 16, families=[(2, 256)])
    k, v = case.keys.cuda(), case.values.cuda()
    table, starts, lengths = case.device_args()
    rows = torch.from_numpy(case.rows).cuda()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    assert tt.paged_attention(case.q.cuda()[:0], k, v, table, starts * 0, lengths, families=rows).shape == (0, 4, 64)
    out = torch.full((2, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    tt.paged_attention(case.q.cuda(), k, v, table[:0], ints(0), ints(), out=out, families=rows[:0])
    tt.paged_attention(case.q.cuda(), k, v, table, ints(0, 0, 0), lengths, out=out, families=rows)
    tt.paged_attention(case.q.cuda(), k, v, table, ints(0, 0, 0), lengths, out=out, window=5, sinks=2)
    assert (out == 7).all()
    for kw in (dict(families=rows), dict(window=3, sinks=2)):
        tt.paged_attention(case.q.cuda(), k, v, table[:, :0].contiguous(), ints(0, 1, 2), ints(0, 0), causal=False, out=out, **kw)
        assert (out == 0).all()
        out.fill_(7)
    tt.cxx.synchronize()


def test_python_refusals_with_device_tensors():
    case = Sight("f16", [1, 3], [300, 290], 4, 2, 64, 16, families=[(2, 256)])
    k, v, q = case.keys.cuda(), case.values.cuda(), case.q.cuda()
    ints = case.device_args()
    rows = torch.from_numpy(case.rows).cuda()
    for bad in (dict(families=rows.long()), dict(families=rows[:1]), dict(families=rows[:, :2]), dict(families=rows.t()), dict(families=rows.cpu()), dict(families=rows[0]),
                dict(families=rows, family_count=-1), dict(families=rows, max_shared=-1), dict(sinks=-1), dict(window=-1, sinks=1), dict(families=rows, scale=0.0)):
        with pytest.raises(tt.cxx.EnforceNotMet):
            tt.paged_attention(q, k, v, *ints, **bad)
    qkv = torch.zeros(case.tokens, 8, 64, dtype=torch.float16, device="cuda")
    norm = torch.ones(64, dtype=torch.float16, device="cuda")
    for bad in (dict(q_norm=norm[:32]), dict(q_norm=norm.cpu()), dict(k_norm=norm.int()), dict(q_norm=norm.view(1, 64)), dict(k_norm=norm.expand(4, 64)),
                dict(q_norm=norm, k_norm=norm.float()), dict(q_norm=norm.bfloat16()), dict(q_norm=norm, eps=-1.0), dict(q_norm=norm, eps=math.nan),
                dict(q_norm=norm, eps=math.inf), dict(q_norm=k.view(-1)[:64]), dict(q_norm=torch.ones(128, dtype=torch.float16, device="cuda")[::2])):
        with pytest.raises(tt.cxx.EnforceNotMet):
            tt.rotary_append(qkv, k, v, *ints, **bad)
    with pytest.raises(tt.cxx.EnforceNotMet):
        tt.rotary_append(qkv, k, v, *ints, inv_freq=tt.rotary_frequencies(64), interleaved=True, q_norm=torch.ones(65, dtype=torch.float16, device="cuda")[1:])


# ------------------------------------------------------------------------------------------------ norms of heads ------
def normed(x, weight, eps):
    """x [.., d] in 64 bits -> (normed, tolerance).

    The tolerance, relative to the result: the sum of squares of d numbers in fp32 (d + 8) 2^-24, 1 / d and its product with it and the sum with eps 3 2^-24, of which the
    root takes half; root, division and two products 5 2^-24."""
    d = x.shape[-1]
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight
    return y, ((d + 11) / 2 + 5) * E32 * y.abs()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 64), (128, 128), (64, 32), (128, 20), (80, 80), (96, 0), (48, 2), (256, 254), (16, 16), (256, 0)])
@pytest.mark.parametrize("which", ["both", "q", "k", "per head"])
def test_rotary_append_with_norms(dt, interleaved, d, rotary, which):
    """Heads of very different sizes, slots besides the new tokens' untouched, values as they were."""
    heads, kv_heads, page = 6, 2, 16
    case = Case(dt, [1, 5, 0, 40], [7, 0, 9, 30], heads, kv_heads, d, page, spare_rows=2)
    gen = torch.Generator().manual_seed(1)
    sizes = torch.tensor([1.0, 1e-3, 30.0, 0.1, 1.0, 5.0, 1e-2, 20.0, 1.0, 1.0])[:, None]
    qkv = (torch.randn(case.tokens, heads + 2 * kv_heads, d, generator=gen) * sizes).to(TORCH_DTYPES[dt])
    eps = 1e-5
    kinds = [torch.float32] if dt == "f32" else [torch.float32, TORCH_DTYPES[dt]]
    inv_freq = tt.rotary_frequencies(rotary, device="cpu", stretch=2.0)
    for kind in kinds:
        shape = lambda n: (n, d) if which == "per head" else (d,)
        weights = [(1 + 0.3 * torch.randn(shape(n), generator=gen)).to(kind) for n in (heads, kv_heads)]
        args = {"q_norm": weights[0].cuda() if which != "k" else None, "k_norm": weights[1].cuda() if which != "q" else None}
        keys, values = case.keys.cuda(), case.values.cuda()
        out = torch.full((case.tokens, heads, d), 7.0, dtype=qkv.dtype, device="cuda")
        q = tt.rotary_append(qkv.cuda(), keys, values, *case.device_args(), inv_freq.cuda(), interleaved, 1.25, out, eps=eps, **args)
        tt.cxx.synchronize()
        n = int(case.starts[-1])
        position = torch.cat([torch.arange(length - m, length) for length, m in zip(case.lengths, case.new)])
        x = qkv[:n, :heads + kv_heads].double()
        y, off = x.clone(), torch.zeros_like(x)
        if which != "k":
            y[:, :heads], off[:, :heads] = normed(x[:, :heads], weights[0].double(), eps)
        if which != "q":
            y[:, heads:], off[:, heads:] = normed(x[:, heads:], weights[1].double(), eps)
        want, tol = turned(y, position, inv_freq, interleaved, 1.25)
        # what the norm is off by goes through the turn: at most the sum of both of a pair, times the amplitude
        through = off.clone()
        i = torch.arange(rotary // 2)
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
        both = 1.25 * (off[..., first] + off[..., second])
        through[..., first], through[..., second] = both, both
        tol = tol + through * (1 + 2 ** -10) + EPS[dt] / 2 * want.abs() * (1 + 2 ** -10) + (2.0 ** -25 if dt == "f16" else 0)
        assert ((q[:n].cpu().double() - want[:, :heads]).abs() <= tol[:, :heads]).all()
        assert (q[n:] == 7).all()
        keys, values = keys.cpu(), values.cpu()
        want_keys, want_values = case.keys.double(), case.values.clone()
        tol_keys = torch.zeros_like(want_keys)
        row = 0
        for b, m in enumerate(case.new):
            for i in range(case.lengths[b] - m, case.lengths[b]):
                at = case.table[b, i // page], slice(None), i % page
                want_keys[at], tol_keys[at], want_values[at] = want[row, heads:], tol[row, heads:], qkv[row, heads + kv_heads:]
                row += 1
        assert torch.equal(values.nan_to_num(nan=99.0), want_values.nan_to_num(nan=99.0))
        assert torch.equal(torch.isnan(keys), torch.isnan(want_keys))
        assert ((keys.double() - want_keys).abs().nan_to_num() <= tol_keys).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 4, 2), (9, 4, 2), (3, 200, 1), (70, 3, 3)])
def test_norms_in_place_and_from_rows_that_lie_apart(dt, tokens, heads, kv_heads):
    """Queries turned where they lie, rows and weights of any alignment: the bits of a call with tensors of their own where the sum's order is the same, else within the
    tolerance."""
    case = Case(dt, [tokens], [30], heads, kv_heads, 64, 16)
    inv_freq = tt.rotary_frequencies(64)
    width = (heads + 2 * kv_heads) * 64
    wide = torch.randn(tokens, width + 128, generator=torch.Generator().manual_seed(3)).to(TORCH_DTYPES[dt]).cuda()
    weight = torch.rand(200 * 64 + 1, generator=torch.Generator().manual_seed(4)).to(TORCH_DTYPES[dt]).cuda()
    for first, off in ((0, 0), (1, 0), (64, 1)):
        qkv = wide[:, first:first + width]
        q_norm, k_norm = weight[off:off + heads * 64].view(heads, 64), weight[off:off + 64]
        keys, values = [case.keys.cuda() for _ in range(2)], [case.values.cuda() for _ in range(2)]
        q = tt.rotary_append(qkv, keys[0], values[0], *case.device_args(), inv_freq, q_norm=q_norm, k_norm=k_norm)
        x, tol = normed(qkv.cpu().double().view(tokens, -1, 64)[:, :heads], q_norm.cpu().double(), 1e-6)
        want, more = turned(x, torch.arange(30, 30 + tokens), inv_freq.cpu(), False, 1.0)
        both = tol[..., :32] + tol[..., 32:]
        tol = torch.cat((both, both), -1) * (1 + 2 ** -10) + more + EPS[dt] / 2 * want.abs() * (1 + 2 ** -10) + (2.0 ** -25 if dt == "f16" else 0)
        assert ((q.cpu().double() - want).abs() <= tol).all()
        kept = wide.clone()
        inside = kept[:, first:first + width]
        tt.rotary_append(inside, keys[1], values[1], *case.device_args(), inv_freq, out=inside[:, :heads * 64], q_norm=q_norm, k_norm=k_norm)
        assert torch.equal(inside[:, :heads * 64], q.view(tokens, heads * 64))
        assert torch.equal(inside[:, heads * 64:], qkv[:, heads * 64:])
        assert torch.equal(keys[0].nan_to_num(), keys[1].nan_to_num()) and torch.equal(values[0].nan_to_num(), values[1].nan_to_num())
    tt.cxx.synchronize()


@pytest.mark.parametrize("dt", DTYPES)
def test_norms_of_zeros_and_of_what_is_not_finite(dt):
    """A head of zeros stays zeros, without eps it is NaN; a NaN or an infinity stays in its head; eps alone of a head far smaller."""
    case = Case(dt, [1, 2], [7, 30], 4, 2, 64, 16)
    keys, values = case.keys.cuda(), case.values.cuda()
    norm = torch.ones(64, device="cuda")
    qkv = torch.randn(3, 8, 64, generator=torch.Generator().manual_seed(3)).to(TORCH_DTYPES[dt]).cuda()
    clean = tt.rotary_append(qkv, keys, values, *case.device_args(), q_norm=norm, k_norm=norm)
    qkv[0, 1] = 0
    qkv[1, 0, 5], qkv[2, 3, 0] = math.nan, math.inf
    got = tt.rotary_append(qkv, keys, values, *case.device_args(), q_norm=norm, k_norm=norm)
    assert (got[0, 1] == 0).all() and torch.isnan(got[1, 0]).all() and torch.isnan(got[2, 3, 0]) and (got[2, 3, 1:] == 0).all()
    for row, head in ((0, 1), (1, 0), (2, 3)):
        got[row, head] = clean[row, head]
    assert torch.equal(got, clean)
    got = tt.rotary_append(qkv, keys, values, *case.device_args(), q_norm=norm, k_norm=norm, eps=0.0)
    assert torch.isnan(got[0, 1]).all() and torch.isfinite(got[0, [0, 2, 3]]).all()
    qkv[0, 2] = 2.0 ** -20
    got = tt.rotary_append(qkv, keys, values, *case.device_args(), q_norm=norm, k_norm=norm, eps=1.0)
    assert ((got[0, 2].double() / 2.0 ** -20 - 1).abs() <= EPS[dt] + 30 * E32).all()


# -------------------------------------------------------------------------------------------------------- together ------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 150)])
def test_a_decoder_whose_samples_share_their_prompt(dt, window, sinks):
    """A prompt, samples of it that grow apart, one of them refused tokens, a fork of a fork, a second prompt among them, a compaction: the context of every step, made with
    `share`, is that of the sequence's own tokens; heads are normed on their way into the cache."""
    layers, heads, kv_heads, d, page = 2, 4, 2, 64, 16
    dtype = TORCH_DTYPES[dt]
    cache = tt.PagedCache(layers, kv_heads, d, 80, page, dtype)
    inv_freq = tt.rotary_frequencies(d)
    gen = torch.Generator().manual_seed(5)
    norms = [[1 + 0.2 * torch.randn(n, d, generator=gen) for n in (heads, kv_heads)] for _ in range(layers)]
    told, families = {}, []

    def step(names, tokens):
        batch = cache.extend(names, tokens, share=True)
        families.append(batch.family_count)
        batch.family_count = batch.max_shared = 0  # (so few keys are read once only where it is not known how few they are)
        for layer in range(layers):
            qkv = torch.randn(sum(tokens), heads + 2 * kv_heads, d, generator=gen).to(dtype)
            at = 0
            for name, n in zip(names, tokens):
                told[name][layer].extend(qkv[at:at + n])
                at += n
            q = cache.append(layer, qkv.cuda(), batch, inv_freq, q_norm=norms[layer][0].cuda(), k_norm=norms[layer][1].cuda())
            got = cache.attend(layer, q, batch, window=window, sinks=sinks).cpu().double()
            at = 0
            for name, n in zip(names, tokens):
                if n:
                    rows = torch.stack(told[name][layer]).double()
                    length = rows.shape[0]
                    y, _ = normed(rows[:, :heads + kv_heads], torch.cat(norms[layer]).double(), 1e-6)
                    y, _ = turned(y, torch.arange(length), inv_freq.cpu(), False, 1.0)
                    y = y.to(dtype).double()
                    key, position = torch.arange(length)[None], torch.arange(length - n, length)[:, None]
                    hidden = key > position
                    if window:
                        hidden |= (key <= position - window) & (key >= sinks)
                    for h in range(heads):
                        s = (y[length - n:, h] @ y[:, heads + h // 2].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                        v = rows[:, heads + kv_heads + h // 2]
                        want = torch.softmax(s, 1) @ v
                        # half a step of q, k and the result each, of the probabilities twice; scores of size 8 at most take the error of q and k
                        bound = (EPS[dt] * 12 + 400 * E32) * max(1.0, float(v.abs().max()))
                        assert (got[at:at + n, h] - want).abs().max() <= bound, (name, layer, h)
                at += n

    def new():
        name = cache.add()
        told[name] = [[] for _ in range(layers)]
        return name

    def fork(name):
        other = cache.fork(name)
        told[other] = [list(rows) for rows in told[name]]
        return other

    a, z = new(), new()
    step([a, z], [200, 150])
    b, c = fork(a), fork(a)
    step([a, b, c, z], [1, 1, 1, 1])
    y = fork(z)
    step([a, b, c, z, y], [1, 40, 3, 1, 1])
    e = fork(b)
    step([c, a, b, e, y, z], [1, 1, 1, 1, 0, 1])
    cache.truncate(b, 205)
    told[b] = [rows[:205] for rows in told[b]]
    cache.free(a)
    cache.compact()
    step([c, b, e, z, y], [1, 2, 1, 30, 1])
    assert families == [0, 1, 2, 2, 2]
    tt.cxx.synchronize()


@pytest.mark.parametrize("dt", DTYPES)
def test_families_and_none_agree(dt):
    """The same batch with and without its families: both within the tolerance of the formula, and what has no family has the same bits as in a call where nobody has."""
    case = Sight(dt, [1] * 9, [700 + 40 * i for i in range(8)] + [400], 8, 2, 128, 16, families=[(8, 640), (1, 0)])
    plain = Case.run_attention(case)
    case.check_attention(plain)
    case.check_attention(case.run_attention())
    assert torch.equal(case.run_attention(hints=None), plain)  # (too few keys to gain anything)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new,window,sinks", [(1, 0, 0), (1, 900, 40), (6, 0, 0)])
def test_families_that_are_worth_it(dt, new, window, sinks):
    """As many common keys as are read once where all is known: those of 70 sequences, cut and joined, and the same bits without hints."""
    rng = random.Random(new)
    past = [2048 + rng.choice([1, 20, 300]) for _ in range(70)] + [900]
    case = Sight(dt, [new] * 71, past, 8, 4, 64, 16, families=[(70, 2048), (1, 0)])
    case.keys, case.values = case.keys.nan_to_num(), case.values.nan_to_num()
    got = case.run_attention(hints=None, window=window, sinks=sinks)
    case.check_attention(got, window=window, sinks=sinks)


def workspace(case, hints, window=0, sinks=0, families=True):
    """What the call of `case` asks for as its workspace: with the families shared it is another one than without."""
    lib = capi.load()
    count, most = hints
    cache = capi.PagedCache(16, 32, *case.keys.shape)  # (addresses that are not looked at)
    batch = capi.PagedBatch(16, case.table.shape[1], 16, 16, len(case.new), case.tokens)
    sight = capi.PagedSight(window, sinks, 16 if families else None, count, most)
    n = ctypes.c_int64(-1)
    dtype = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[case.dt]
    capi.check(lib.ttmi_paged_attention_sight_workspace(ctypes.byref(cache), ctypes.byref(batch), case.heads, max(case.new), max(case.lengths), ctypes.byref(sight), dtype,
                                                        ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new,keys,window,sinks", [(1, 2048, 0, 0), (1, 2048, 2000, 40), (20, 4096, 0, 0)])
def test_shared_and_not_shared_by_the_hints(dt, new, keys, window, sinks):
    """A batch whose hints let its families be shared, and one that they do not, by the workspace that the call asks for: both, and the calls without hints, which share, and without
    families give every sequence the formula's results; what is not shared has the bits of a call without families."""
    rng = random.Random(new)
    many = Sight(dt, [new] * 71, [keys + rng.choice([1, 20, 300]) for _ in range(70)] + [900], 8, 4, 64, 16, families=[(70, keys), (1, 0)])
    few = Sight(dt, [new] * 5, [150 + 9 * i for i in range(4)] + [200], 8, 4, 64, 16, families=[(4, 144), (1, 0)])
    for case, hints, shared in ((many, (1, keys), True), (few, (1, 144), False)):
        kw = dict(window=window, sinks=sinks)
        assert (workspace(case, hints, **kw) != workspace(case, hints, families=False, **kw)) == shared
        assert workspace(case, (0, 0), **kw) != workspace(case, (0, 0), families=False, **kw)
        hinted, unknown, none = case.run_attention(hints=None, **kw), case.run_attention(**kw), Case.run_attention(case, **kw)
        want, tol = case.attention(**kw)
        for got in (hinted, unknown, none):
            assert ((got.cpu().double() - want).abs() <= tol).all()
        assert shared or torch.equal(hinted, none)
