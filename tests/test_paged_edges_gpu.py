"""Attention over pages where scores, values and queries are infinite, not numbers or very large, in every way that the work is cut; and long prompts side by side."""
import math

import pytest
import torch

import turbotransformers_amd as tt
from test_paged_gpu import DTYPES, Case, check

pytestmark = pytest.mark.gpu

# (new tokens, keys before them in 16-bit types and in fp32, heads, kv_heads, head_dim): which kernel works on the sequences, and which one joins their parts
WAYS = {
    "few rows, whole": ([1, 3], [200, 90], [200, 90], 4, 2, 64),
    "few rows, joined by row": ([1, 3], [5000, 3000], [5000, 3000], 4, 2, 64),
    "few rows of many, joined by row": ([1] * 40, [2500 + 7 * i for i in range(40)], [1500 + 7 * i for i in range(40)], 4, 2, 64),
    "few rows, joined by pair": ([1] * 64, [1500, 1700] + [100 + i for i in range(62)], [1500, 1700] + [100 + i for i in range(62)], 16, 8, 64),
    "tiles, whole": ([30, 60], [20, 10], [20, 10], 4, 2, 128),
    "tiles, two parts": ([20], [492], [108], 48, 12, 64),
    "tiles, some parts": ([20], [3000], [800], 4, 2, 64),
    "tiles, many parts": ([20], [9000], [2500], 4, 1, 128),
}


def made(way, dt, **kw):
    new, past16, past32, heads, kv_heads, d = WAYS[way]
    return Case(dt, new, past32 if dt == "f32" else past16, heads, kv_heads, d, 16, **kw)


def slot(case, b, key):
    return int(case.table[b, key // case.page]), slice(None), key % case.page


def rows_of(case, b):
    return range(int(case.starts[b]), int(case.starts[b + 1]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("way", WAYS)
def test_rows_whose_scores_are_all_minus_infinity(dt, way):
    """Zero divided by zero is NaN; zeros are for tokens that see no key.  The first element of every key is 1, that of one query minus infinity: its other heads and the
    other tokens have what they have without it."""
    case = made(way, dt)
    case.keys[..., 0] = torch.where(torch.isnan(case.keys[..., 0]), case.keys[..., 0], torch.ones_like(case.keys[..., 0]))
    clean = case.run_attention()
    case.check_attention(clean)
    hit = [(rows_of(case, b)[0], 1) for b in range(len(case.new))] + [(rows_of(case, len(case.new) - 1)[-1], 2)]
    for row, head in hit:
        case.q[row, head, 0] = -math.inf
    got = case.run_attention()
    for row, head in hit:
        assert torch.isnan(got[row, head]).all(), (row, head)
        got[row, head] = clean[row, head]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("way", WAYS)
def test_keys_of_weight_zero(dt, way):
    """Scores of minus infinity among others, the first keys' of a sequence among them: the bits of scores so low that their weights are zero."""
    case = made(way, dt)
    case.q[..., 0] = 8.0  # times -60000 and a scale of at least 128^-1/2: 2^-60000 and less is 0
    hit = [(b, key) for b, n in enumerate(case.lengths) for key in [*range(10), n // 2]]
    for b, key in hit:
        case.keys[slot(case, b, key)][..., 0] = -60000.0
    low = case.run_attention()
    case.check_attention(low)
    for b, key in hit:
        case.keys[slot(case, b, key)][..., 0] = -math.inf
    assert torch.equal(case.run_attention(), low)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("way", WAYS)
def test_the_largest_values(dt, way):
    """Values of one sign whose sum over a token's keys is just below 2^120, where every weight but the first tile's is 2^7.9 before the division: no sum leaves fp32, and
    the mean of equal values is that value."""
    case = made(way, dt)
    case.q.zero_()
    case.q[..., 0] = 8.0
    kept = torch.isnan(case.keys)
    case.keys.zero_()
    for b, n in enumerate(case.lengths):
        for key in range(16, n):
            case.keys[slot(case, b, key)][..., 0] = 7.9 * math.log(2) * math.sqrt(case.d) / 8
    case.keys[kept] = math.nan
    value = 2.0 ** (119 - math.ceil(math.log2(max(case.lengths)))) * 1.875
    case.values = torch.where(torch.isnan(case.values), case.values, torch.full_like(case.values, value))
    case.check_attention(case.run_attention())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("way", WAYS)
def test_what_is_not_finite_stays_with_the_rows_that_see_it(dt, bad, way):
    """A value of the last key/value head, at the first key, in the middle, at the first new token and at the last: NaN (or an infinity) in its column for the tokens that
    see it, the same bits as without it everywhere else.  A query's element: NaN in its own row and head."""
    case = made(way, dt)
    clean = case.run_attention()
    case.check_attention(clean)
    kept, group = case.values.clone(), case.heads // case.kv_heads
    for where in (lambda n, m: 0, lambda n, m: (n - m) // 2, lambda n, m: n - m, lambda n, m: n - 1):
        case.values.copy_(kept)
        spoiled = torch.zeros(case.q.shape, dtype=torch.bool)
        for b, (n, m) in enumerate(zip(case.lengths, case.new)):
            key = where(n, m)
            case.values[slot(case, b, key)][-1, 7] = bad
            for row in rows_of(case, b):
                spoiled[row, case.heads - group:, 7] = n - m + row - rows_of(case, b)[0] >= key
        got = case.run_attention().cpu()
        assert torch.equal(torch.isnan(got) if math.isnan(bad) else ~torch.isfinite(got), spoiled)
        assert torch.equal(got[~spoiled], clean.cpu()[~spoiled])
    case.values.copy_(kept)
    spoiled = torch.zeros(case.q.shape, dtype=torch.bool)
    for b in range(len(case.new)):
        case.q[rows_of(case, b)[-1], 1, 5] = bad
        spoiled[rows_of(case, b)[-1], 1] = True
    got = case.run_attention().cpu()
    assert torch.equal(torch.isnan(got), spoiled)
    assert torch.equal(got[~spoiled], clean.cpu()[~spoiled])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("way", WAYS)
def test_an_infinite_value_behind_a_weight_of_zero(dt, bad, way):
    """Its key has a score so low that its weight is zero: an infinity or NaN for those who see it (which one is not said), in its column alone."""
    case = made(way, dt)
    case.q[..., 0] = 8.0
    for b, n in enumerate(case.lengths):
        case.keys[slot(case, b, 3)][..., 0] = -60000.0
    clean = case.run_attention().cpu()
    for b in range(len(case.new)):
        case.values[slot(case, b, 3)][0, 9] = bad
    spoiled = torch.zeros(case.q.shape, dtype=torch.bool)
    spoiled[:, :case.heads // case.kv_heads, 9] = True
    got = case.run_attention().cpu()
    assert torch.equal(~torch.isfinite(got), spoiled)
    assert torch.equal(got[~spoiled], clean[~spoiled])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window", [0, 400])
def test_prompts_of_many_blocks_side_by_side(dt, window):
    """More workgroups than the chip takes at a time: they begin with the sequences of most keys, in these with the last rows; single tokens among them."""
    case = Case(dt, [300, 1, 1500, 700, 1, 1100, 513], [0, 90, 7, 200, 0, 0, 33], 24, 12, 64, 16, spare_rows=1)
    case.check_attention(case.run_attention(window=window), window=window)


@pytest.mark.parametrize("dt", DTYPES)
def test_a_sequence_alone_and_among_others(dt):
    """How the work is cut depends on the whole batch, so bits may differ; both are within the tolerance of the formula."""
    case = Case(dt, [1, 40, 1, 300, 7], [3000, 100, 17, 0, 900], 8, 2, 128, 16)
    together = case.run_attention()
    want, tol = case.attention()
    keys, values, (table, _, lengths) = case.keys.cuda(), case.values.cuda(), case.device_args()
    for b, n in enumerate(case.new):
        rows = slice(int(case.starts[b]), int(case.starts[b + 1]))
        alone = tt.paged_attention(case.q[rows].cuda(), keys, values, table[b:b + 1], torch.tensor([0, n], dtype=torch.int32, device="cuda"), lengths[b:b + 1],
                                   max_tokens=n, max_length=case.lengths[b])
        for got in (alone, together[rows]):
            assert ((got.cpu().double() - want[rows]).abs() <= tol[rows]).all(), b
    tt.cxx.synchronize()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window", [0, 6000])
def test_long_contexts_beside_prompts(dt, window):
    """Few tokens over thousands of keys, cut and joined, in one call with a prompt and a chunk behind many keys; sequences without new tokens among them."""
    check(dt, [1, 700, 3, 0, 90], [9000, 0, 5000, 70, 3000], 8, 2, 64, 16, window=window, spare_rows=1)
