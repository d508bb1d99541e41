"""The book of a cache in pages, and what the operators over such a cache refuse.  No GPU."""
import ctypes
import random

import numpy as np
import pytest
import torch

import turbotransformers_amd as tt
from turbotransformers_amd import capi


# ------------------------------------------------------------------------------------------------------ the book ------
class Memory:
    """What the slots of a cache would hold: (sequence's own history) written through the book alone."""

    def __init__(self, pool):
        self.pool, self.slots = pool, {}

    def move(self, pairs):
        to = [p[1] for p in pairs]
        assert len(set(to)) == len(to) and not set(to) & {p[0] for p in pairs}
        old = dict(self.slots)
        for src, dst in pairs:
            for i in range(self.pool.page_size):
                self.slots[dst, i] = old.get((src, i))

    def write(self, sequence, position, value):
        pages = self.pool.pages_of(sequence)
        self.slots[pages[position // self.pool.page_size], position % self.pool.page_size] = value

    def read(self, sequence):
        pages, size = self.pool.pages_of(sequence), self.pool.page_size
        return [self.slots.get((pages[i // size], i % size)) for i in range(self.pool.length(sequence))]


@pytest.mark.parametrize("page_size", [1, 4, 16])
@pytest.mark.parametrize("seed", range(4))
def test_pool_keeps_every_sequence_whatever_the_others_do(page_size, seed):
    """Random adds, forks, growth, truncation, frees and compactions: every sequence reads back what was written to it, no page
    has another count than the sequences that hold it, and none is lost."""
    rng = random.Random(seed)
    pool = tt.cxx.PagePool(60, page_size)
    memory, held, mark = Memory(pool), {}, 0
    for _ in range(400):
        what = rng.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        if what == "add" and len(held) < 12:
            held[pool.add()] = []
        elif what == "extend" and held:
            names = rng.sample(sorted(held), rng.randint(1, len(held)))
            tokens = [rng.choice([0, 1, 1, 2, 7]) for _ in names]
            before = {n: (pool.pages_of(n), pool.length(n)) for n in held}
            try:
                copies = pool.extend(names, tokens)
            except tt.cxx.EnforceNotMet:
                assert before == {n: (pool.pages_of(n), pool.length(n)) for n in held}
                continue
            memory.move(copies)
            for name, n in zip(names, tokens):
                for _ in range(n):
                    mark += 1
                    memory.write(name, len(held[name]), mark)
                    held[name].append(mark)
        elif what == "fork" and held and len(held) < 12:
            name = rng.choice(sorted(held))
            held[pool.fork(name)] = list(held[name])
        elif what == "truncate" and held:
            name = rng.choice(sorted(held))
            n = rng.randint(0, len(held[name]))
            pool.truncate(name, n)
            held[name] = held[name][:n]
        elif what == "free" and len(held) > 3:
            name = rng.choice(sorted(held))
            pool.free(name)
            del held[name]
        elif what == "compact":
            memory.move(pool.compact())
            used = {p for name in held for p in pool.pages_of(name)}
            assert used == set(range(len(used)))
        counts = {}
        for name in held:
            assert pool.length(name) == len(held[name])
            assert len(pool.pages_of(name)) == -(-len(held[name]) // page_size)
            assert memory.read(name) == held[name]
            for page in pool.pages_of(name):
                counts[page] = counts.get(page, 0) + 1
        assert [pool.references(p) for p in range(60)] == [counts.get(p, 0) for p in range(60)]
        assert pool.free_pages == 60 - len(counts)
        assert pool.sequences == len(held)


def test_pool_copies_a_shared_page_once_less_than_it_is_shared():
    pool = tt.cxx.PagePool(10, 4)
    a = pool.add()
    assert pool.extend([a], [6]) == []
    b, c = pool.fork(a), pool.fork(a)
    shared = pool.pages_of(a)
    copies = pool.extend([a, b, c], [1, 1, 1])
    assert [src for src, _ in copies] == [shared[1]] * 2
    assert len({pool.pages_of(s)[1] for s in (a, b, c)}) == 3
    assert [pool.pages_of(s)[0] for s in (a, b, c)] == [shared[0]] * 3


def test_pool_does_not_copy_a_full_page():
    pool = tt.cxx.PagePool(10, 4)
    a = pool.add()
    pool.extend([a], [8])
    b = pool.fork(a)
    assert pool.extend([a, b], [1, 1]) == []
    assert pool.pages_of(a)[:2] == pool.pages_of(b)[:2] and pool.pages_of(a)[2] != pool.pages_of(b)[2]


def test_pool_refuses():
    for args in ((-1, 16), (4, 0), (4, 3), (4, 8192)):
        with pytest.raises(tt.cxx.EnforceNotMet):
            tt.cxx.PagePool(*args)
    pool = tt.cxx.PagePool(2, 4)
    a = pool.add()
    for call in (lambda: pool.extend([a], [9]), lambda: pool.extend([a, a], [1, 1]), lambda: pool.extend([a], [-1]), lambda: pool.extend([a], [1, 2]),
                 lambda: pool.extend([a + 1], [1]), lambda: pool.fork(7), lambda: pool.free(7), lambda: pool.truncate(a, 1), lambda: pool.references(2),
                 lambda: pool.references(-1), lambda: pool.length(7)):
        with pytest.raises(tt.cxx.EnforceNotMet):
            call()
    pool.extend([a], [8])
    with pytest.raises(tt.cxx.EnforceNotMet):
        pool.table([a], 1)
    np.testing.assert_array_equal(pool.table([a], 3), [pool.pages_of(a) + [0]])
    assert pool.table([], 3).shape == (0, 3)


def test_pool_says_beforehand_what_it_will_copy_and_move():
    """`copies_of` and `moves_of` change nothing, name what `extend` and `compact` then return, and refuse what `extend` refuses."""
    rng = random.Random(1)
    pool = tt.cxx.PagePool(30, 4)
    held = [pool.add()]
    book = lambda: [(s, pool.pages_of(s), pool.length(s)) for s in held] + [pool.free_pages] + [pool.references(p) for p in range(30)]
    seen = 0
    for _ in range(300):
        names = rng.sample(held, rng.randint(1, len(held)))
        tokens = [rng.choice([0, 1, 2, 7]) for _ in names]
        before = book()
        try:
            copies = pool.copies_of(names, tokens)
        except tt.cxx.EnforceNotMet:
            assert book() == before
            with pytest.raises(tt.cxx.EnforceNotMet):
                pool.extend(names, tokens)
            assert book() == before
            for s in held[1:]:
                pool.free(s)
            held = held[:1]
            pool.truncate(held[0], rng.randint(0, 9))
            continue
        assert book() == before
        free = {p for p in range(30) if pool.references(p) == 0}
        assert {to for _, to in copies} <= free
        assert pool.extend(names, tokens) == copies
        seen += len(copies)
        if len(held) < 6:
            held.append(pool.fork(rng.choice(held)))
        if rng.random() < 0.2:
            before, moves = book(), pool.moves_of()
            assert book() == before
            assert {to for _, to in moves} <= {p for p in range(30) if pool.references(p) == 0}
            assert pool.compact() == moves
            seen += len(moves)
    assert seen > 50


class FailsOnce(Exception):
    pass


@pytest.mark.parametrize("fails", ["copy", "batch"])
def test_a_step_that_cannot_be_made_leaves_the_sequences_as_they_were(fails, monkeypatch):
    """The copy of a shared page is refused (here: memory of the host), or the batch cannot be built: every sequence has its tokens as before, and the same
    call made again copies the page."""
    from turbotransformers_amd.layers import paged
    cache = tt.PagedCache(1, 1, 16, 8, 4, torch.float32, device="cpu")
    a = cache.add()
    cache.extend([a], [6])
    b = cache.fork(a)
    shared = cache.pool.pages_of(a)[1]
    held = lambda: [(cache.pool.length(s), cache.pool.pages_of(s)[0]) for s in (a, b)]
    before, copied = held(), []
    if fails == "copy":
        with pytest.raises(tt.cxx.EnforceNotMet, match="not on the GPU"):
            cache.extend([a, b], [1, 7])
        assert cache.pool.pages_of(a) == cache.pool.pages_of(b) and cache.pool.free_pages == 6
    monkeypatch.setattr(paged, "copy_pages", lambda keys, values, src, dst: copied.extend(zip(src, dst)))
    if fails == "batch":
        def no_batch(*args):
            raise FailsOnce
        with monkeypatch.context() as m:
            m.setattr(paged, "PagedBatch", no_batch)
            with pytest.raises(FailsOnce):
                cache.extend([a, b], [1, 7])
    assert held() == before
    batch = cache.extend([a, b], [1, 7])
    assert [cache.length(s) for s in (a, b)] == [7, 13] and batch.lengths.tolist() == [7, 13] and batch.starts.tolist() == [0, 1, 8]
    last = [cache.pool.pages_of(s)[1] for s in (a, b)]
    assert last[0] != last[1] and len(copied) == 1 and copied[0][0] == shared and copied[0][1] in last


def test_a_compaction_that_cannot_be_made_changes_nothing(monkeypatch):
    from turbotransformers_amd.layers import paged
    cache = tt.PagedCache(1, 1, 16, 8, 4, torch.float32, device="cpu")
    a, b = cache.add(), cache.add()
    cache.extend([a, b], [9, 5])
    cache.free(a)
    book = lambda: (cache.pool.pages_of(b), cache.pool.free_pages, [cache.pool.references(p) for p in range(8)])
    before = book()
    with pytest.raises(tt.cxx.EnforceNotMet, match="not on the GPU"):
        cache.compact()
    assert book() == before
    moved = []
    monkeypatch.setattr(paged, "copy_pages", lambda keys, values, src, dst: moved.extend(zip(src, dst)))
    assert cache.compact() == 2 and [src for src, _ in moved] == before[0] and cache.pool.pages_of(b) == [0, 1]


# ----------------------------------------------------------------------------------------------------- refusals ------
P = ctypes.c_void_p
ADDRESS = 1 << 20  # (nothing is read: every call below is refused before a launch)


def cache(**changes):
    fields = dict(keys=ADDRESS, values=ADDRESS, pages=4, kv_heads=2, page_size=16, head_dim=64)
    fields.update(changes)
    return capi.PagedCache(**fields)


def batch(**changes):
    fields = dict(table=ADDRESS, table_pitch=2, starts=ADDRESS, lengths=ADDRESS, batch=2, tokens=3)
    fields.update(changes)
    return capi.PagedBatch(**fields)


def append(ttmi, c, b, qkv=ADDRESS, qkv_pitch=512, q=2 * ADDRESS, q_pitch=256, heads=4, inv_freq=ADDRESS, rotary=64, interleaved=0, dtype=capi.F16):
    return ttmi.ttmi_rotary_append(P(qkv), qkv_pitch, P(q), q_pitch, heads, ctypes.byref(c) if c else None, ctypes.byref(b) if b else None, P(inv_freq), rotary,
                                   interleaved, 1.0, dtype, None)


def attend(ttmi, c, b, q=ADDRESS, q_pitch=256, out=2 * ADDRESS, out_pitch=256, heads=4, max_tokens=0, max_length=0, scale=0.125, window=0, workspace=None,
           bytes=0, dtype=capi.F16):
    return ttmi.ttmi_paged_attention(P(q), q_pitch, P(out), out_pitch, heads, ctypes.byref(c) if c else None, ctypes.byref(b) if b else None, max_tokens,
                                     max_length, scale, 1, window, P(workspace), bytes, dtype, None)


BAD_CACHE = [dict(page_size=0), dict(page_size=24), dict(page_size=8192), dict(head_dim=0), dict(head_dim=72), dict(head_dim=272), dict(kv_heads=0),
             dict(kv_heads=3), dict(pages=-1), dict(keys=None), dict(values=None), dict(keys=ADDRESS + 8), dict(values=ADDRESS + 2)]
BAD_BATCH = [dict(table=None), dict(starts=None), dict(lengths=None), dict(batch=-1), dict(tokens=-1), dict(table_pitch=-1), dict(table_pitch=1 << 30),
             dict(table_pitch=(1 << 26) + 1), dict(tokens=1 << 23)]


@pytest.fixture(scope="module")
def lib():
    return capi.load()


@pytest.mark.parametrize("call", [append, attend])
def test_bad_caches_and_batches_are_refused(lib, call):
    for changes in BAD_CACHE:
        assert call(lib, cache(**changes), batch()) == -1, changes
        assert lib.ttmi_last_error()
    for changes in BAD_BATCH:
        assert call(lib, cache(), batch(**changes)) == -1, changes
    assert call(lib, None, batch()) == -1 and call(lib, cache(), None) == -1
    for changes in (dict(heads=0), dict(heads=3), dict(dtype=capi.I8), dict(dtype=17)):
        assert call(lib, cache(), batch(), **changes) == -1, changes


@pytest.mark.parametrize("call", [append, attend])
def test_tables_whose_slots_pass_64_bits_are_refused(lib, call):
    """table_pitch * page_size of 2^64, 2^63 and 2^52 + 1 times 4096, of which 64 bits hold 0, a negative number and 4096."""
    for pitch, size in ((1 << 52, 4096), (1 << 51, 4096), ((1 << 52) + 1, 4096), ((1 << 60) + 4, 16), ((1 << 63) - 1, 2)):
        assert call(lib, cache(page_size=size), batch(table_pitch=pitch)) == -1, (pitch, size)


def test_append_refuses(lib):
    for changes in (dict(qkv=None), dict(q=None), dict(inv_freq=None), dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(qkv_pitch=511), dict(q_pitch=255),
                    dict(q=ADDRESS), dict(qkv=ADDRESS + 1), dict(qkv=ADDRESS + 2, interleaved=1)):
        assert append(lib, cache(), batch(), **changes) == -1, changes
    # nothing to do
    assert append(lib, cache(), batch(tokens=0)) == 0 and append(lib, cache(), batch(batch=0)) == 0


def test_attention_refuses(lib):
    for changes in (dict(q=None), dict(out=None), dict(q=ADDRESS + 8), dict(out=ADDRESS + 2), dict(q_pitch=252), dict(q_pitch=258), dict(out_pitch=260),
                    dict(window=-1), dict(max_tokens=-1), dict(max_length=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                    dict(scale=float("nan"))):
        assert attend(lib, cache(), batch(), **changes) == -1, changes
    for d in (16, 80, 96, 256):
        assert attend(lib, cache(head_dim=d), batch(), q_pitch=4 * d, out_pitch=4 * d) == -1
    assert attend(lib, cache(), batch(tokens=0)) == 0 and attend(lib, cache(), batch(batch=0)) == 0
    n = ctypes.c_int64(-7)
    assert lib.ttmi_paged_attention_workspace(ctypes.byref(cache(page_size=3)), ctypes.byref(batch()), 4, 0, 0, 0, capi.F16, ctypes.byref(n)) == -1
    assert lib.ttmi_paged_attention_workspace(ctypes.byref(cache()), ctypes.byref(batch()), 4, 0, 0, 0, capi.F16, None) == -1


def test_scales_whose_product_with_log2_e_is_not_finite_are_refused(lib):
    """The kernels multiply scores by scale * log2(e), 1.4427 of it: 2.3585e38 * 1.4427 is below the largest fp32 number 3.4028e38, 2.3587e38 * 1.4427 is above."""
    for scale in (2.3587e38, 2.5e38, 3e38, 3.4e38):
        assert attend(lib, cache(), batch(), scale=scale) == -1, scale
        assert b"scale" in lib.ttmi_last_error()
    assert attend(lib, cache(), batch(tokens=0), scale=2.3585e38) == 0


def test_launches_that_are_too_large_are_refused(lib):
    """Before anything is started: more rows, or more sequences, than a launch has threads for."""
    assert attend(lib, cache(kv_heads=1), batch(tokens=1 << 20), heads=1 << 10, q_pitch=1 << 16, out_pitch=1 << 16) == -1
    assert attend(lib, cache(), batch(batch=1 << 22)) == -1
    assert copy(lib, [0], [1], page_bytes=(1 << 36) + 16) == -1


@pytest.mark.parametrize("dtype", [capi.F32, capi.F16])
def test_workspace_does_not_grow_with_keys_that_a_window_hides(lib, dtype):
    """What 300 tokens see of their last 500 keys, cut into parts: as much room with a table for 2^24 positions as with one for 2^12 (and some at all)."""
    sizes = []
    for pitch in (1 << 8, 1 << 20):
        n = ctypes.c_int64(-7)
        assert lib.ttmi_paged_attention_workspace(ctypes.byref(cache(pages=1 << 20)), ctypes.byref(batch(batch=1, tokens=300, table_pitch=pitch)), 4, 300, 0, 500,
                                                  dtype, ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] == sizes[1] and 0 < sizes[0] <= 300 * 4 * 66 * 4 * 20


@pytest.mark.parametrize("dtype", [capi.F32, capi.F16])
@pytest.mark.parametrize("tokens", [1, 300])
def test_workspace_of_a_window_that_hides_nothing(lib, dtype, tokens):
    """However far a window reaches beyond the longest context, to the largest number there is: the same cut (one that needs room)."""
    sizes = []
    for window in (1 << 22, 1 << 30, (1 << 31) + 5, (1 << 63) - 1 - tokens, (1 << 63) - 1):
        n = ctypes.c_int64(-7)
        assert lib.ttmi_paged_attention_workspace(ctypes.byref(cache(pages=1 << 20)), ctypes.byref(batch(batch=1, tokens=tokens, table_pitch=1 << 12)), 4, tokens, 0,
                                                  window, dtype, ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert len(set(sizes)) == 1 and sizes[0] > 0, sizes


@pytest.mark.parametrize("dtype", [capi.F32, capi.F16, capi.BF16])
def test_long_contexts_beside_a_prompt_are_shared_out(lib, dtype):
    """Single tokens over 100000 keys and a prompt that fills the chip by itself: room for the parts that their keys are cut into.  The prompt alone, prompts of one
    length and short contexts beside a prompt need none."""
    def room(sequences, tokens, most, longest):
        n = ctypes.c_int64(-7)
        assert lib.ttmi_paged_attention_workspace(ctypes.byref(cache(pages=1 << 20, kv_heads=8, head_dim=128)),
                                                  ctypes.byref(batch(batch=sequences, tokens=tokens, table_pitch=1 << 14)), 32, most, longest, 0, dtype,
                                                  ctypes.byref(n)) == 0
        return n.value
    assert room(9, 4104, 4096, 100000) > 0
    assert room(2, 4097, 4096, 100000) > 0
    assert room(1, 4096, 4096, 100000) == 0
    assert room(3, 12288, 4096, 100000) == 0
    assert room(9, 4104, 4096, 1000) == 0


def copy(ttmi, sources, destinations, keys=ADDRESS, values=ADDRESS, layers=1, pages=8, page_bytes=64):
    a, b = (np.asarray(x, np.int32) for x in (sources, destinations))
    return ttmi.ttmi_copy_pages(P(keys), P(values), layers, pages, page_bytes, P(a.ctypes.data), P(b.ctypes.data), len(a), None)


def test_copies_of_pages_that_are_refused(lib):
    for src, dst in (([0], [8]), ([8], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([0, 2, 4], [1, 3, 0])):
        assert copy(lib, src, dst) == -1, (src, dst)
    for changes in (dict(keys=None), dict(values=None), dict(keys=ADDRESS + 8), dict(layers=-1), dict(layers=40000), dict(page_bytes=24), dict(page_bytes=-16)):
        assert copy(lib, [0], [1], **changes) == -1, changes
    assert copy(lib, [], []) == 0 and copy(lib, [0], [1], layers=0) == 0


def test_python_calls_that_are_refused():
    """Tensors of the host, of other types and shapes, and no tensors at all."""
    kv = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    ints = [torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)]
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.float16)
    for call in (lambda: tt.paged_attention(q, kv, kv.clone(), *ints), lambda: tt.rotary_append(qkv, kv, kv.clone(), *ints),
                 lambda: tt.copy_pages(kv, kv.clone(), [0], [1])):
        with pytest.raises(tt.cxx.EnforceNotMet, match="not on the GPU"):
            call()
    with pytest.raises(tt.cxx.EnforceNotMet, match="expected a tensor"):
        tt.paged_attention(q, kv, 3, *ints)
    with pytest.raises(ValueError):
        tt.rotary_append(qkv[:, :256], kv, kv, *ints)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=4, stretch=0.0), dict(rotary_dim=4, trained_length=100, slow_turns=3.0, fast_turns=2.0)):
        with pytest.raises(ValueError):
            tt.rotary_frequencies(**bad, device="cpu")


def test_rotary_frequencies():
    f = tt.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64
    np.testing.assert_allclose(f.numpy(), [1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    np.testing.assert_allclose(tt.rotary_frequencies(8, 100.0, 4.0, device="cpu").numpy(), f.numpy() / 4, rtol=1e-15)
    # 2 pi * 10 tokens: pair i makes 10 f_i turns; 1 (kept from 8 on), in between, and stretched below 2
    g = tt.rotary_frequencies(8, 100.0, 4.0, trained_length=62.83185307179586, slow_turns=2.0, fast_turns=8.0, device="cpu")
    kept = np.clip((10 * f.numpy() - 2) / 6, 0, 1)
    np.testing.assert_allclose(g.numpy(), f.numpy() * (kept + (1 - kept) / 4), rtol=1e-14)
    assert g[0] == f[0] and 0 < kept[1] < 1
    np.testing.assert_allclose(g[2:].numpy(), f[2:].numpy() / 4, rtol=1e-14)
    assert tt.rotary_frequencies(0, device="cpu").numel() == 0
