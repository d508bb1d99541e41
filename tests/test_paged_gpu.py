"""Rotary append, attention over pages and page copies against the formulas in 64 bits."""
import ctypes
import math
import random

import numpy as np
import pytest
import torch

import turbotransformers_amd as tt
from helpers import TORCH_DTYPES
from turbotransformers_amd import capi

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]
EPS = {dt: torch.finfo(TORCH_DTYPES[dt]).eps for dt in DTYPES}
E32 = 2.0 ** -24  # half a step of fp32


class Case:
    """A batch over a cache whose unused slots, pages and rows hold NaN (or, where they are read as numbers, a marker)."""

    def __init__(self, dt, new, past, heads, kv_heads, d, page, seed=0, spare_rows=0, spare_width=0, scale_q=1.0):
        gen = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.dt, self.d, self.page, self.heads, self.kv_heads = dt, d, page, heads, kv_heads
        self.new, self.lengths = list(new), [n + p for n, p in zip(new, past)]
        need = [-(-n // page) for n in self.lengths]
        pages = sum(need) + 3
        order = rng.sample(range(pages), sum(need))
        self.table = np.full((len(new), max(need + [1]) + spare_width), 1 << 30, np.int32)  # behind the last page: not to be read
        for b, n in enumerate(need):
            self.table[b, :n] = [order.pop() for _ in range(n)]
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.starts[-1]) + spare_rows
        dtype = TORCH_DTYPES[dt]
        shape = (pages, kv_heads, page, d)
        self.keys, self.values = torch.full(shape, math.nan), torch.full(shape, math.nan)
        for b, n in enumerate(self.lengths):
            for i in range(n):
                self.keys[self.table[b, i // page], :, i % page] = torch.randn(kv_heads, d, generator=gen)
                self.values[self.table[b, i // page], :, i % page] = torch.randn(kv_heads, d, generator=gen)
        self.keys, self.values = self.keys.to(dtype), self.values.to(dtype)
        self.q = (torch.randn(self.tokens, heads, d, generator=gen) * scale_q).to(dtype)
        self.q[int(self.starts[-1]):] = math.nan

    def device_args(self):
        return [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (self.table, self.starts, self.lengths)]

    def history(self, b, cache):
        """[length, kv_heads, d] in 64 bits."""
        n = self.lengths[b]
        pages = self.table[b, :-(-n // self.page)].tolist()
        return cache[pages].transpose(1, 2).reshape(-1, self.kv_heads, self.d)[:n].double()

    def attention(self, causal=True, window=0, scale=None):
        """-> (out, tolerance) [tokens, heads, d], NaN behind the last sequence.

        The tolerance, for a score s = scale sum_i q_i k_i, o = sum_j p_j v_j and a = sum_j p_j |v_j|:
        scores: d products and sums in fp32, the scale, the argument of the exponential and its last places: each |s| error is at most
          ds = (d + 6) 2^-24 scale sum_i |q_i k_i|, as is that of the maximum; p changes by 2 ds in proportion, the sum likewise: 4 ds a;
        sums over n keys in fp32: 2 (n + 8) 2^-24 a (numerator and denominator);
        probabilities rounded to 16 bits for the product with v: half a step each, in numerator and (summed as rounded or not) denominator: eps a; fp16 ones
          below its least normal number besides by at most 2^-25 each, against a sum of at least 1: n 2^-25 max |v| twice;
        partial results joined: 8 2^-24 a; the result rounded: eps / 2 |o|."""
        scale = scale if scale is not None else 1 / math.sqrt(self.d)
        eps = EPS[self.dt]
        out = torch.full((self.tokens, self.heads, self.d), math.nan, dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        for b, n in enumerate(self.lengths):
            k, v = self.history(b, self.keys), self.history(b, self.values)
            rows = slice(int(self.starts[b]), int(self.starts[b + 1]))
            m = rows.stop - rows.start
            if m == 0:
                continue
            position = torch.arange(n - m, n)[:, None]
            key = torch.arange(n)[None]
            hidden = torch.zeros(m, n, dtype=torch.bool)
            if causal:
                hidden |= key > position
            if window:
                hidden |= key <= position - window
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

    def check_attention(self, got, **kw):
        want, tol = self.attention(**kw)
        got = got.cpu().double().reshape(want.shape)
        n = int(self.starts[-1])
        assert not torch.isnan(got[:n]).any()
        worst = ((got[:n] - want[:n]).abs() - tol[:n]).max() if n else torch.tensor(-1.0)
        assert worst <= 1e-30, "over the tolerance by %g at %s" % (worst, np.unravel_index(((got - want).abs() - tol)[:n].argmax(), want[:n].shape))
        return want

    def run_attention(self, out=None, max_tokens=None, max_length=None, **kw):
        args = self.device_args()
        out = torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device="cuda") if out is None else out
        hints = dict(max_tokens=max(self.new) if max_tokens is None else max_tokens, max_length=max(self.lengths) if max_length is None else max_length)
        got = tt.paged_attention(self.q.cuda(), self.keys.cuda(), self.values.cuda(), *args, out=out, **hints, **kw)
        tt.cxx.synchronize()
        torch.cuda.synchronize()
        return got


def check(dt, new, past, heads, kv_heads, d, page, causal=True, window=0, scale=None, **kw):
    case = Case(dt, new, past, heads, kv_heads, d, page, **kw)
    got = case.run_attention(causal=causal, window=window, scale=scale)
    case.check_attention(got, causal=causal, window=window, scale=scale)
    assert (got[int(case.starts[-1]):] == 7.0).all()  # rows behind the last sequence are left as they were


# --------------------------------------------------------------------------------------------------- attention ------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (8, 1), (16, 2)])
def test_single_tokens(dt, d, heads, kv_heads):
    """Decoding: lengths of one to several tiles, at and around their edges, a page that ends inside a tile; spare rows behind the batch."""
    lengths = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 257]
    check(dt, [1] * len(lengths), [n - 1 for n in lengths], heads, kv_heads, d, 16, spare_rows=3)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(2, 2, 16), (6, 2, 32), (8, 1, 64), (32, 2, 16)])
def test_chunks(dt, d, heads, kv_heads, page):
    """Prompts and chunks of every size around the tiles' edges, single tokens and sequences without new tokens among them."""
    new = [1, 3, 0, 16, 17, 33, 65, 130]
    past = [40, 0, 9, 100, 0, 31, 64, 5]
    check(dt, new, past, heads, kv_heads, d, page, spare_rows=2, spare_width=1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page", [1, 2, 8, 16, 128, 256, 4096])
def test_page_sizes(dt, page):
    check(dt, [1, 20, 1], [70, 50, 290], 4, 2, 64, page)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 50, 64, 100, 10000])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(dt, window, causal):
    check(dt, [1, 90, 1, 7], [300, 40, 0, 129], 4, 2, 128, 16, causal=causal, window=window)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_windows_over_long_contexts_are_cut_and_joined(dt, causal):
    """Few blocks of rows whose windows begin and end anywhere in the parts that their keys are cut into; more keys than was said; a window longer than some."""
    for window, new, past in ((1000, [40], [5000]), (700, [130, 9, 20], [2999, 100, 4000]), (2000, [20], [1500])):
        check(dt, new, past, 4, 2, 64, 16, causal=causal, window=window, spare_rows=1)
    case = Case(dt, [90, 30], [3000, 17], 4, 2, 64, 16)
    case.check_attention(case.run_attention(max_tokens=30, max_length=400, window=900, causal=causal), window=900, causal=causal)


@pytest.mark.parametrize("dt", DTYPES)
def test_all_keys_are_seen_without_causality(dt):
    check(dt, [1, 70, 3], [5, 30, 200], 4, 2, 64, 16, causal=False)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_long_contexts_are_cut_and_joined(dt, d):
    """A few tokens over thousands of keys, beside short ones."""
    check(dt, [1, 1, 5], [5000, 3, 2500], 4, 1, d, 32)
    check(dt, [1], [9000], 2, 2, d, 16)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (1 << 30, 1 << 40), (3, 100)])
def test_hints_choose_nothing_but_the_cut(dt, hints):
    case = Case(dt, [1, 40, 1], [600, 100, 30], 8, 2, 64, 16)
    case.check_attention(case.run_attention(max_tokens=hints[0], max_length=hints[1]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("scale", [1e-4, 1.0, 3.0])
def test_scales(dt, scale):
    check(dt, [1, 40], [200, 100], 4, 2, 64, 16, scale=scale)


@pytest.mark.parametrize("dt", DTYPES)
def test_tokens_that_see_no_key(dt):
    """An empty memory (no causality, no keys), and more new tokens than keys: zeros."""
    case = Case(dt, [2, 3, 1], [5, 0, 0], 4, 2, 64, 16)
    case.lengths[1] = 0
    got = case.run_attention(causal=False).cpu()
    assert (got[2:5] == 0).all()
    case.check_attention(got, causal=False)
    case = Case(dt, [20, 1], [0, 40], 4, 2, 64, 16)
    case.lengths[0] = 7  # its 20 tokens have positions -13 to 6
    got = case.run_attention(max_length=41).cpu()
    assert (got[:13] == 0).all()
    torch.testing.assert_close(got[13].view(2, 2, 64)[:, 0], case.values[case.table[0, 0], :, 0])  # sees the first key alone


@pytest.mark.parametrize("dt", DTYPES)
def test_values_and_scores_far_from_zero(dt):
    """Keys whose scores lie hundreds apart, one infinite value behind a zero probability, a NaN behind the token's own position."""
    case = Case(dt, [1, 30], [150, 70], 4, 2, 64, 16, scale_q=30.0)
    case.check_attention(case.run_attention())
    case = Case(dt, [30], [70], 4, 2, 64, 16)
    page, slot = case.table[0, 99 // 16], 99 % 16
    case.keys[page, :, slot] = math.nan
    case.values[page, :, slot] = math.nan
    got = case.run_attention()
    assert torch.isnan(got[29]).all()
    case.keys[page, :, slot], case.values[page, :, slot] = 0, 0
    case.q[29] = 0
    case.check_attention(torch.cat((got[:29], case.run_attention()[29:])))


@pytest.mark.parametrize("dt", DTYPES)
def test_rows_that_lie_apart(dt):
    """q as part of a wider tensor, out as part of another, two-dimensional ones."""
    case = Case(dt, [1, 20], [100, 7], 4, 2, 64, 16)
    wide = torch.zeros(case.tokens, 8 * 64, dtype=case.q.dtype, device="cuda")
    wide[:, 64:64 + 256] = case.q.cuda().view(-1, 256)
    result = torch.full((case.tokens, 512), 7.0, dtype=case.q.dtype, device="cuda")
    got = tt.paged_attention(wide[:, 64:320], case.keys.cuda(), case.values.cuda(), *case.device_args(), out=result[:, 128:384])
    case.check_attention(got)
    assert (result[:, :128] == 7).all() and (result[:, 384:] == 7).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_reaches_only_the_tokens_that_see_it(dt, bad):
    """One value of a key of each of three sequences, one decoding, one with a few rows, one with many: rows whose windows and positions leave that key out
    have what they would have without it, the others a NaN or an infinity in that column alone; and a query of it spoils its own rows only."""
    new, past, window = [1, 5, 150], [300, 290, 200], 100
    case = Case(dt, new, past, 4, 2, 64, 16)
    clean = case.run_attention(window=window)
    case.check_attention(clean, window=window)
    hit = [[280, 0], [193, 260], [250, 149]]  # (seen by all or only by some of the new tokens, or behind the window)
    kept = case.values.clone()
    for which in range(2):
        case.values.copy_(kept)
        for b in range(3):
            case.values[case.table[b, hit[b][which] // 16], 1, hit[b][which] % 16, 7] = bad
        got = case.run_attention(window=window)
        for b in range(3):
            for i in range(new[b]):
                row, position = int(case.starts[b]) + i, past[b] + i
                sees = position - window < hit[b][which] <= position
                spoiled = torch.zeros(4, 64, dtype=torch.bool)
                spoiled[2:, 7] = sees
                assert torch.equal(~torch.isfinite(got[row]).cpu(), spoiled), (which, b, i)
                assert torch.equal(got[row].cpu()[~spoiled], clean[row].cpu()[~spoiled]), (which, b, i)
    case.values.copy_(kept)
    for row in (0, 3, 70):
        case.q[row, 2, 5] = bad
    got = case.run_attention(window=window)
    for row in range(sum(new)):
        spoiled = [row in (0, 3, 70) and h == 2 for h in range(4)]
        for h in range(4):
            if spoiled[h]:
                assert torch.isnan(got[row, h]).all(), row
            else:
                assert torch.equal(got[row, h], clean[row, h]), (row, h)


def test_result_does_not_depend_on_what_else_is_in_the_batch_or_runs_twice():
    """The same call twice gives the same bits, in every type, cut or not."""
    for dt in DTYPES:
        case = Case(dt, [1, 40, 1], [3000, 100, 17], 8, 2, 128, 16)
        assert torch.equal(case.run_attention(), case.run_attention())


@pytest.mark.parametrize("dt", DTYPES)
def test_offsets_beyond_32_bits(dt):
    """A cache of more than 2^32 bytes (2^31 elements in 16-bit types) whose last pages are read and written."""
    d, page, kv_heads = 128, 64, 8
    pages = (1 << 31) // (kv_heads * page * d) + 40
    keys = torch.zeros((pages, kv_heads, page, d), dtype=TORCH_DTYPES[dt], device="cuda")
    values = torch.zeros_like(keys)
    case = Case(dt, [1, 20], [100, 37], 16, kv_heads, d, page)
    used = sorted({int(p) for row, n in zip(case.table, case.lengths) for p in row[:-(-n // page)]})
    high = {p: pages - 1 - i for i, p in enumerate(used)}
    for p, h in high.items():
        keys[h], values[h] = case.keys[p].cuda(), case.values[p].cuda()
    table = torch.tensor([[high.get(int(p), 0) for p in row] for row in case.table], dtype=torch.int32, device="cuda")
    _, starts, lengths = case.device_args()
    got = tt.paged_attention(case.q.cuda(), keys, values, table, starts, lengths, max_length=200)
    case.check_attention(got)
    qkv = torch.randn(case.tokens, 32, d, device="cuda").to(keys.dtype)
    tt.rotary_append(qkv, keys, values, table, starts, lengths)
    last = int(table[1, (case.lengths[1] - 1) // page])
    assert torch.equal(values[last, :, (case.lengths[1] - 1) % page], qkv[-1, 24:])
    tt.copy_pages(keys, values, [last], [pages - 40])
    assert torch.equal(keys[pages - 40].nan_to_num(), keys[last].nan_to_num()) and torch.equal(values[pages - 40].nan_to_num(), values[last].nan_to_num())
    tt.cxx.synchronize()


def test_pages_outside_the_cache_are_reported():
    case = Case("f16", [1, 30], [100, 7], 4, 2, 64, 16)
    case.keys, case.values = case.keys.nan_to_num(), case.values.nan_to_num()
    for bad in (-1, 1 << 20):
        table, starts, lengths = case.device_args()
        table[0, 2] = bad
        for call in (lambda: tt.paged_attention(case.q.cuda(), case.keys.cuda(), case.values.cuda(), table, starts, lengths),):
            out = call()
            torch.cuda.synchronize()
            with pytest.raises(tt.cxx.EnforceNotMet, match="out of range"):
                tt.cxx.synchronize()
            tt.cxx.synchronize()  # reported once
            good = torch.cat((case.run_attention()[:1], out[1:]))
            case.check_attention(good)  # the other sequence
        table[0, 100 // 16] = bad
        keys, values = case.keys.cuda(), case.values.cuda()
        tt.rotary_append(torch.ones(case.tokens, 8, 64, dtype=torch.float16, device="cuda"), keys, values, table, starts, lengths)
        torch.cuda.synchronize()
        with pytest.raises(tt.cxx.EnforceNotMet, match="out of range"):
            tt.cxx.synchronize()
        untouched = [p for p in range(keys.shape[0]) if p not in case.table[1]]
        assert torch.equal(keys[untouched].cpu(), case.keys[untouched])
    # more keys than the table has pages for: those there are
    table, starts, lengths = case.device_args()
    lengths[0] = 5000
    tt.paged_attention(case.q.cuda(), case.keys.cuda(), case.values.cuda(), table[:, :7].contiguous(), starts, lengths)
    torch.cuda.synchronize()
    with pytest.raises(tt.cxx.EnforceNotMet, match="out of range"):
        tt.cxx.synchronize()


# ------------------------------------------------------------------------------------------------------ append ------
def turned(x, position, inv_freq, interleaved, amplitude):
    """x [tokens, heads, d] and positions in 64 bits -> (turned, tolerance before the rounding to the type).

    The tolerance: sine and cosine in fp32, a rounded argument of at most pi/4 (2^-25) and sums of at most 1 with two roundings that count (2 2^-24), times an
    amplitude rounded once more: 4 2^-24 of each; two products, of which one is rounded, and a sum: 2 2^-24 (|x1| + |x2|)."""
    r = 2 * len(inv_freq)
    y, tol = x.clone(), torch.zeros_like(x)
    i = torch.arange(r // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    angle = (position.double()[:, None] * inv_freq)[:, None]
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    x1, x2 = x[..., first], x[..., second]
    y[..., first], y[..., second] = x1 * c - x2 * s, x1 * s + x2 * c
    for part in (first, second):
        tol[..., part] = 6 * E32 * amplitude * (x1.abs() + x2.abs())
    return y, tol


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 64), (128, 128), (64, 32), (128, 20), (80, 80), (96, 0), (48, 2), (256, 254), (16, 16)])
def test_rotary_append(dt, interleaved, d, rotary):
    """All heads of the new tokens, slots besides theirs untouched, one past position in the hundreds of thousands' place."""
    heads, kv_heads, page = 6, 2, 16
    case = Case(dt, [1, 5, 0, 40], [7, 0, 9, 30], heads, kv_heads, d, page, spare_rows=2)
    gen = torch.Generator().manual_seed(1)
    qkv = torch.randn(case.tokens, heads + 2 * kv_heads, d, generator=gen).to(TORCH_DTYPES[dt])
    inv_freq = tt.rotary_frequencies(rotary, device="cpu", stretch=2.0)
    keys, values = case.keys.cuda(), case.values.cuda()
    out = torch.full((case.tokens, heads, d), 7.0, dtype=qkv.dtype, device="cuda")
    q = tt.rotary_append(qkv.cuda(), keys, values, *case.device_args(), inv_freq.cuda(), interleaved, 1.25, out)
    tt.cxx.synchronize()
    n = int(case.starts[-1])
    position = torch.cat([torch.arange(length - m, length) for length, m in zip(case.lengths, case.new)])
    want, tol = turned(qkv[:n, :heads + kv_heads].double(), position, inv_freq, interleaved, 1.25)
    tol = tol + EPS[dt] / 2 * want.abs() * (1 + 2 ** -10)
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
    if rotary == 0:
        assert torch.equal(q[:n].cpu(), qkv[:n, :heads])


@pytest.mark.parametrize("dt", DTYPES)
def test_rotary_positions_far_out(dt):
    """Positions up to 10^6 and beyond: the angle of the fastest pair is the position itself."""
    d, heads = 64, 2
    for past in (0, 131071, 1 << 20, 16000000):
        width = (past + 2) // 4096 + 1
        table = torch.full((1, width), 0, dtype=torch.int32, device="cuda")
        keys = torch.zeros(1, 1, 4096, d, dtype=TORCH_DTYPES[dt], device="cuda")
        values = torch.zeros_like(keys)
        qkv = torch.randn(2, heads + 2, d, generator=torch.Generator().manual_seed(past)).to(keys.dtype)
        inv_freq = tt.rotary_frequencies(d, device="cpu")
        q = tt.rotary_append(qkv.cuda(), keys, values, table, torch.tensor([0, 2], dtype=torch.int32, device="cuda"),
                             torch.tensor([past + 2], dtype=torch.int32, device="cuda"), inv_freq.cuda())
        want, tol = turned(qkv[:, :heads].double(), torch.arange(past, past + 2), inv_freq, False, 1.0)
        assert ((q.cpu().double() - want).abs() <= tol + EPS[dt] / 2 * want.abs() * (1 + 2 ** -10)).all(), past
    tt.cxx.synchronize()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens", [1, 9])
def test_append_in_place_and_from_rows_that_lie_apart(dt, tokens):
    """Queries turned where they lie, in rows of a wider tensor: the same bits as into a tensor of their own."""
    case = Case(dt, [tokens], [30], 4, 2, 64, 16)
    inv_freq = tt.rotary_frequencies(64)
    wide = torch.randn(tokens, 10 * 64, generator=torch.Generator().manual_seed(3)).to(TORCH_DTYPES[dt]).cuda()
    for first in (0, 1, 64):  # (1: rows that are not aligned to 16 bytes)
        qkv = wide[:, first:first + 512]
        keys, values = [case.keys.cuda() for _ in range(2)], [case.values.cuda() for _ in range(2)]
        q = tt.rotary_append(qkv, keys[0], values[0], *case.device_args(), inv_freq)
        kept = wide.clone()
        inside = kept[:, first:first + 512]
        assert tt.rotary_append(inside, keys[1], values[1], *case.device_args(), inv_freq, out=inside[:, :256]) is not None
        assert torch.equal(inside[:, :256], q.view(tokens, 256))
        assert torch.equal(inside[:, 256:], qkv[:, 256:])
        assert torch.equal(keys[0].nan_to_num(), keys[1].nan_to_num()) and torch.equal(values[0].nan_to_num(), values[1].nan_to_num())
    tt.cxx.synchronize()


# -------------------------------------------------------------------------------------------------------- copies ------
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layers,kv_heads,page,d,count", [(1, 1, 1, 16, 1), (3, 2, 16, 64, 5), (12, 12, 16, 64, 4), (2, 3, 8, 80, 40), (1, 1, 1, 16, 1500)])
def test_copy_pages(dt, layers, kv_heads, page, d, count):
    """Copies in all layers, more of them than one launch takes; one source many times; pages besides the destinations untouched."""
    pages = 2 * count + 3
    gen = torch.Generator("cuda").manual_seed(count)
    keys, values = (torch.randn((layers, pages, kv_heads, page, d), generator=gen, device="cuda").to(TORCH_DTYPES[dt]) for _ in range(2))
    order = random.Random(count).sample(range(pages), 2 * count)
    src, dst = order[:count], order[count:]
    src[1:3] = [src[0]] * len(src[1:3])
    want = [x.clone() for x in (keys, values)]
    for x, w in zip((keys, values), want):
        w[:, dst] = x[:, src]
    tt.copy_pages(keys, values, src, dst)
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])
    tt.copy_pages(keys[0], values[0], [dst[0]], [src[0]])
    assert torch.equal(keys[0, src[0]], keys[0, dst[0]])
    tt.copy_pages(keys, values, [], [])


# -------------------------------------------------------------------------------------------------- refusals on the device ------
def test_python_refusals_with_device_tensors():
    case = Case("f16", [1, 3], [20, 7], 4, 2, 64, 16)
    k, v, q = case.keys.cuda(), case.values.cuda(), case.q.cuda()
    table, starts, lengths = case.device_args()
    attend = lambda **kw: tt.paged_attention(*[{**dict(q=q, k=k, v=v, table=table, starts=starts, lengths=lengths), **kw}[n] for n in
                                               ("q", "k", "v", "table", "starts", "lengths")])
    for bad in (dict(table=table.long()), dict(starts=starts.long()), dict(lengths=lengths.float()), dict(lengths=lengths[:1]), dict(starts=starts[:2]),
                dict(table=table.cpu()), dict(k=k.float()), dict(v=v[:-1]), dict(k=k.transpose(1, 2)), dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.transpose(0, 1)),
                dict(q=q[..., :32]), dict(table=table.t()), dict(k=k.long(), v=v.long())):
        with pytest.raises(tt.cxx.EnforceNotMet):
            attend(**bad)
    with pytest.raises(tt.cxx.EnforceNotMet, match="overlaps"):
        tt.paged_attention(q, k, v, table, starts, lengths, out=q)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(tt.cxx.EnforceNotMet, match="scale"):
            tt.paged_attention(q, k, v, table, starts, lengths, scale=scale)
    qkv = torch.zeros(case.tokens, 8, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(tt.cxx.EnforceNotMet, match="overlaps"):
        tt.rotary_append(qkv, k, v, table, starts, lengths, out=qkv[:, 1:5])
    # memory that a kernel reads and another of its workgroups writes
    inside = k.view(-1)[:q.numel()].view(q.shape)
    for call in (lambda: tt.paged_attention(q, k, v, table, starts, lengths, out=inside), lambda: tt.rotary_append(qkv, k, v, table, starts, lengths, out=inside),
                 lambda: tt.rotary_append(qkv, k, k, table, starts, lengths), lambda: tt.copy_pages(v, v, [0], [1]),
                 lambda: tt.rotary_append(k.view(-1)[:qkv.numel()].view(qkv.shape), k, v, table, starts, lengths)):
        with pytest.raises(tt.cxx.EnforceNotMet, match="overlap"):
            call()
    # tensors of another device than the current one
    for call in (lambda: tt.cxx.paged_attention(q, k, v, table, starts, lengths, torch.empty_like(q), 0, 0, None, True, 0, None, 1, 0),
                 lambda: tt.cxx.rotary_append(qkv, k, v, table, starts, lengths, None, False, 1.0, torch.empty_like(q), 1, 0),
                 lambda: tt.cxx.copy_pages(k, v, [0], [1], 1, 0)):
        with pytest.raises(tt.cxx.EnforceNotMet, match="the current device is 1"):
            call()
    with pytest.raises(tt.cxx.EnforceNotMet):
        tt.rotary_append(qkv, k, v, table, starts, lengths, inv_freq=torch.ones(32, device="cuda"))
    with pytest.raises(tt.cxx.EnforceNotMet):
        tt.copy_pages(k, v, [0], [1, 2])
    with pytest.raises(tt.cxx.EnforceNotMet):
        tt.copy_pages(k.transpose(2, 3), v.transpose(2, 3), [0], [1])
    out = tt.paged_attention(q.detach().requires_grad_(), k, v, table, starts, lengths)  # (inference: gradients are not followed)
    case.check_attention(out)


# -------------------------------------------------------------------------------------------------------- together ------
@pytest.mark.parametrize("dt", DTYPES)
def test_a_decoder_over_a_shared_cache(dt):
    """Prompts in chunks, single tokens, forks that write into a shared page, a truncation, a compaction, page reuse: every step's context is that of the
    sequence's own tokens, as computed from them alone."""
    layers, heads, kv_heads, d, page = 2, 4, 2, 64, 16
    cache = tt.PagedCache(layers, kv_heads, d, 24, page, TORCH_DTYPES[dt])
    inv_freq = tt.rotary_frequencies(d)
    gen = torch.Generator().manual_seed(5)
    told = {}  # sequence -> the rows of Q|K|V of its tokens, [layer][token]

    def step(names, tokens):
        batch = cache.extend(names, tokens)
        for layer in range(layers):
            qkv = torch.randn(sum(tokens), heads + 2 * kv_heads, d, generator=gen).to(TORCH_DTYPES[dt])
            at = 0
            for name, n in zip(names, tokens):
                told[name][layer].extend(qkv[at:at + n])
                at += n
            q = cache.append(layer, qkv.cuda(), batch, inv_freq)
            got = cache.attend(layer, q, batch).cpu().double()
            at = 0
            for name, n in zip(names, tokens):
                if n:
                    rows = torch.stack(told[name][layer]).double()
                    length = rows.shape[0]
                    y, _ = turned(rows[:, :heads + kv_heads], torch.arange(length), inv_freq.cpu(), False, 1.0)
                    y = y.to(TORCH_DTYPES[dt]).double()
                    for h in range(heads):
                        s = y[length - n:, h] @ y[:, heads + h // 2].T / math.sqrt(d)
                        s = s.masked_fill(torch.arange(length)[None] > torch.arange(length - n, length)[:, None], -math.inf)
                        want = torch.softmax(s, 1) @ rows[:, heads + kv_heads + h // 2]
                        # half a step of q, k and the result each, of the probabilities twice; scores of size 8 at most take the error of q and k
                        bound = (EPS[dt] * 12 + 400 * E32) * max(1.0, float(rows[:, heads + kv_heads + h // 2].abs().max()))
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

    a, b = new(), new()
    step([a, b], [37, 5])
    step([b, a], [30, 1])
    c, e = fork(a), fork(a)
    step([a, b, c, e], [1, 1, 1, 1])
    step([c, a, e], [20, 1, 0])
    cache.free(a)
    cache.truncate(c, 40)
    told[c] = [rows[:40] for rows in told[c]]
    f = fork(c)
    step([c, b, f], [1, 2, 9])
    cache.free(e)
    cache.compact()
    step([b, c, f], [1, 33, 1])
    tt.cxx.synchronize()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_recorded_steps(dt):
    """A decoding step recorded into a graph and replayed with growing lengths, eager work on the same cache and synchronisations between the replays; a
    second graph over the same cache, whose workspace is its own, replayed in turn."""
    case = Case(dt, [1, 1, 1], [690, 3, 55], 8, 2, 128, 16, spare_width=3)  # (each sequence's pages have room for four tokens more)
    table, starts, lengths = case.device_args()
    table.clamp_(0, case.keys.shape[0] - 1)
    keys, values = case.keys.nan_to_num().cuda(), case.values.nan_to_num().cuda()
    qkv = torch.randn(3, 12, 128, generator=torch.Generator().manual_seed(2)).to(keys.dtype).cuda()
    inv_freq = tt.rotary_frequencies(128)

    def call():
        q = tt.rotary_append(qkv, keys, values, table, starts, lengths, inv_freq)
        return tt.paged_attention(q, keys, values, table, starts, lengths, max_tokens=1, max_length=720)

    call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for turn in range(4):
        qkv.copy_(torch.randn(3, 12, 128, generator=torch.Generator().manual_seed(10 + turn)).to(keys.dtype))
        lengths.add_(1)
        want = call()
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            out.fill_(math.nan)
            graph.replay()
            torch.randn(1 << 16, device="cuda").sum()
            torch.cuda.synchronize()
            assert torch.equal(out, want), turn
    tt.cxx.synchronize()


def test_two_streams_at_once():
    """Calls on two streams share nothing: both give what each gives alone."""
    cases = [Case("bf16", [1, 1], [4000, 900], 8, 2, 128, 16, seed=s) for s in range(2)]
    args = [[c.q.cuda(), c.keys.cuda(), c.values.cuda(), *c.device_args()] for c in cases]
    want = [tt.paged_attention(*a, max_tokens=1) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tt.paged_attention(*args[i], max_tokens=1))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_c_interface():
    """The same call through the C ABI: the workspace it asks for, and its refusal of a smaller one."""
    lib = capi.load()
    case = Case("f16", [1, 1], [5000, 20], 4, 1, 64, 16)
    q, k, v = case.q.cuda(), case.keys.cuda(), case.values.cuda()
    table, starts, lengths = case.device_args()
    cache = capi.PagedCache(k.data_ptr(), v.data_ptr(), k.shape[0], 1, 16, 64)
    batch = capi.PagedBatch(table.data_ptr(), table.shape[1], starts.data_ptr(), lengths.data_ptr(), 2, 2)
    n = ctypes.c_int64(-1)
    capi.check(lib.ttmi_paged_attention_workspace(ctypes.byref(cache), ctypes.byref(batch), 4, 1, 5001, 0, capi.F16, ctypes.byref(n)))
    assert n.value >= 0
    work = torch.empty(max(16, n.value), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    call = lambda bytes: lib.ttmi_paged_attention(q.data_ptr(), 256, out.data_ptr(), 256, 4, ctypes.byref(cache), ctypes.byref(batch), 1, 5001, 0.125, 1, 0,
                                                  work.data_ptr(), bytes, capi.F16, stream)
    capi.check(call(n.value))
    torch.cuda.synchronize()
    case.check_attention(out)
    assert torch.equal(out, case.run_attention(max_tokens=1, max_length=5001))
    if n.value:
        assert call(n.value - 1) == -1


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("batch", [64, 65, 130, 400])
def test_many_sequences(dt, batch):
    """More sequences than a wavefront has lanes, long ones among short ones, some without new tokens: shared out evenly and joined, and in blocks of many rows."""
    rng = random.Random(batch)
    lengths = [rng.choice([1, 5, 40, 90, 700 if i % 9 == 0 else 130]) for i in range(batch)]
    new = [0 if i % 7 == 3 else 1 for i in range(batch)]
    check(dt, new, [n - m for n, m in zip(lengths, new)], 4, 2, 64, 16, spare_rows=1)
    case = Case(dt, new, [n - m for n, m in zip(lengths, new)], 4, 2, 64, 16, seed=1)
    case.check_attention(case.run_attention(max_length=5000))  # (long enough for sharing out)
    new = [40 if i % 11 == 0 else m for i, m in enumerate(new)]
    check(dt, new, lengths, 4, 2, 64, 16)


@pytest.mark.parametrize("dt", DTYPES)
def test_more_heads_of_a_group_than_rows_of_a_tile(dt):
    check(dt, [1, 3, 2], [20, 5, 300], 200, 1, 64, 16)
    check(dt, [2], [700], 150, 1, 128, 32, window=33)


def test_calls_on_two_streams_at_a_time():
    """Two batches over one cache, cut and joined, in turn on two streams without waiting for one another: their workspaces are their own."""
    cases = [Case("bf16", [1] * 3, [3000, 2000, 900], 8, 2, 128, 16, seed=1), Case("bf16", [40, 1], [2500, 1200], 8, 2, 128, 16, seed=2)]
    tensors = [[x.cuda() for x in (case.q, case.keys, case.values)] + case.device_args() for case in cases]
    hints = [dict(max_tokens=max(case.new), max_length=max(case.lengths)) for case in cases]
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


def test_recorded_copies():
    """The list of a recorded copy is the recording's own: the lists it was given may change, the pages' contents may."""
    keys, values = (torch.randn(2, 30, 2, 16, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    src, dst = [1, 5, 7], [10, 20, 3]
    tt.copy_pages(keys, values, [0], [29])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tt.copy_pages(keys, values, src, dst)
    src[0], dst[0] = 2, 4
    for _ in range(3):
        keys.normal_(), values.normal_()
        want = [x.clone() for x in (keys, values)]
        for w in want:
            w[:, [10, 20, 3]] = w[:, [1, 5, 7]]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(keys, want[0]) and torch.equal(values, want[1])


def test_sequences_without_keys_and_calls_without_tokens():
    """No tokens at all, no sequences, a table without columns for sequences that are empty: nothing is written, nothing goes wrong."""
    case = Case("f16", [1, 1], [20, 3], 4, 2, 64, 16)
    k, v = case.keys.cuda(), case.values.cuda()
    table, starts, lengths = case.device_args()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    assert tt.paged_attention(case.q.cuda()[:0], k, v, table, starts * 0, lengths).shape == (0, 4, 64)
    out = torch.full((2, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    tt.paged_attention(case.q.cuda(), k, v, table[:0], ints(0), ints(), out=out)
    tt.paged_attention(case.q.cuda(), k, v, table, ints(0, 0, 0), lengths, out=out)
    assert (out == 7).all()
    tt.paged_attention(case.q.cuda(), k, v, table[:, :0].contiguous(), ints(0, 1, 2), ints(0, 0), causal=False, out=out)
    assert (out == 0).all()
    qkv = torch.ones(2, 8, 64, dtype=torch.float16, device="cuda")
    before = k.clone()
    assert tt.rotary_append(qkv[:0], k, v, table, starts * 0, lengths).shape == (0, 4, 64)
    tt.rotary_append(qkv, k, v, table, ints(0, 0, 0), lengths)
    assert torch.equal(k.nan_to_num(), before.nan_to_num())
    tt.cxx.synchronize()
