"""Which sequences of a step are a family, and what the append with norms and the attention with families and first tokens refuse.  No GPU."""
import ctypes
import random

import numpy as np
import pytest
import torch

import turbotransformers_amd as tt
from test_paged_cache import ADDRESS, BAD_BATCH, BAD_CACHE, P, batch, cache
from turbotransformers_amd import capi
from turbotransformers_amd.layers import paged


# ---------------------------------------------------------------------------------------------------- families ------
def shared_cache(pages=200, page_size=16):
    return tt.PagedCache(1, 1, 16, pages, page_size, torch.float32, device="cpu")


def test_forks_are_a_family(monkeypatch):
    """What neighbours have in common, in whole pages that were full before the step; a page that forks have come to have of their own is not; others are alone."""
    monkeypatch.setattr(paged, "copy_pages", lambda *args: None)
    c = shared_cache()
    a, z = c.add(), c.add()
    c.extend([a, z], [300, 200])
    b = c.fork(a)
    step = c.extend([a, b, z], [1, 2, 1], share=True)
    assert step.families.tolist() == [[0, 2, 288], [0, 2, 288], [2, 3, 0]] and step.families.dtype == torch.int32
    assert (step.family_count, step.max_shared) == (1, 288)
    assert step.lengths.tolist() == [301, 302, 201] and step.starts.tolist() == [0, 1, 3, 4]
    assert c.extend([a, z, b], [0, 0, 0], share=True).families is None  # not neighbours
    assert c.extend([a, b, z], [1, 1, 1]).families is None  # not asked for
    y = c.fork(z)
    step = c.extend([y, z, b, a], [50, 0, 1, 1], share=True)
    assert step.families.tolist() == [[0, 2, 192]] * 2 + [[2, 4, 288]] * 2 and (step.family_count, step.max_shared) == (2, 288)


def test_tokens_of_the_step_are_not_shared(monkeypatch):
    """Sequences in common pages that this very step fills: only what was full before counts."""
    monkeypatch.setattr(paged, "copy_pages", lambda *args: None)
    c = shared_cache()
    a = c.add()
    c.extend([a], [256])
    b = c.fork(a)
    c.truncate(b, 130)
    assert c.extend([a, b], [1, 1], share=True).families.tolist() == [[0, 2, 128]] * 2
    c.truncate(b, 127)
    assert c.extend([a, b], [1, 100], share=True).families is None


def test_a_family_takes_a_further_member_where_that_saves_keys():
    """Three texts that begin alike: rows of pages 0..99 in common by 100, 100, then 20 pages.  Two members more of the short prefix are worth it, one is not."""
    def rows(*common):  # common[i]: pages of 8 slots that i and i + 1 begin with
        pool = tt.cxx.PagePool(1000, 8)
        names = [pool.add()]
        pool.extend(names, [800])
        for n in common:
            names.append(pool.fork(names[-1]))
            pool.truncate(names[-1], 8 * n)
            pool.extend(names[-1:], [800 - 8 * n])
        return pool.families(names, [800] * len(names), 128)
    got, count, most = rows(100, 100, 20)
    assert got.tolist() == [[0, 3, 800]] * 3 + [[3, 4, 0]] and (count, most) == (1, 800)
    got, count, most = rows(30, 20)  # 2 * 160 > 240
    assert got.tolist() == [[0, 3, 160]] * 3 and (count, most) == (1, 160)
    got, count, most = rows(50, 20, 50)  # 2 * 160 < 400: two pairs
    assert got.tolist() == [[0, 2, 400]] * 2 + [[2, 4, 400]] * 2 and (count, most) == (2, 400)
    got, count, most = rows(15, 0, 16)  # 120 keys are too few
    assert got.tolist() == [[0, 1, 0], [1, 2, 0], [2, 4, 128], [2, 4, 128]] and (count, most) == (1, 128)


@pytest.mark.parametrize("seed", range(6))
def test_families_are_runs_with_the_same_pages(seed, monkeypatch):
    """Random forks and growth: every row names a run that holds its sequence, all of it says the same, and the pages it promises are the same and full."""
    monkeypatch.setattr(paged, "copy_pages", lambda *args: None)
    rng = random.Random(seed)
    size = rng.choice([1, 16, 64])
    c = shared_cache(8000 // size * 8, size)
    held, seen = [c.add()], 0
    c.extend(held, [rng.randint(100, 700)])
    for _ in range(40):
        if len(held) < 14:
            held.insert(rng.randrange(len(held) + 1), c.fork(rng.choice(held)) if rng.random() < 0.8 else c.add())
        if rng.random() < 0.3:
            name = rng.choice(held)
            c.truncate(name, rng.randint(0, c.length(name)))
        before = [c.length(s) for s in held]
        step = c.extend(held, [rng.choice([0, 1, 1, 40]) for _ in held], share=True)
        if step.families is None:
            assert step.family_count == step.max_shared == 0
            continue
        rows, table = step.families.tolist(), step.table.tolist()
        keys = {row[0]: row[2] for row in rows if row[2]}
        assert step.family_count == len(keys) and step.max_shared == max(keys.values())
        for b, (first, end, n) in enumerate(rows):
            assert first <= b < end <= len(held) and rows[first] == rows[b] and n % size == 0
            assert (n == 0) == (end - first == 1) and (n == 0 or n >= 128) and n <= before[b]
            assert table[b][:n // size] == table[first][:n // size]
        seen += step.family_count
    assert seen > 20


def test_families_refuse():
    pool = tt.cxx.PagePool(10, 4)
    a = pool.add()
    for call in (lambda: pool.families([a], [], 1), lambda: pool.families([a + 1], [1], 1)):
        with pytest.raises(tt.cxx.EnforceNotMet):
            call()
    pool.extend([a], [8])
    b = pool.fork(a)
    # (never more than a sequence has, whatever is said)
    assert pool.families([a, b], [100, -5], 1)[1:] == (0, 0) and pool.families([a, b], [100, 100], 1)[0].tolist() == [[0, 2, 8]] * 2
    assert pool.families([], [], 1)[0].shape == (0, 3)


def test_a_step_without_sequences_or_tokens():
    c = shared_cache()
    assert c.extend([], [], share=True).families is None
    a = c.add()
    assert c.extend([a], [0], share=True).families is None
    assert c.extend([a, c.fork(a)], [0, 0], share=True).families is None


# ---------------------------------------------------------------------------------------------------- refusals ------
@pytest.fixture(scope="module")
def lib():
    return capi.load()


def append(ttmi, c, b, qkv=ADDRESS, qkv_pitch=512, q=2 * ADDRESS, q_pitch=256, heads=4, inv_freq=ADDRESS, rotary=64, interleaved=0, dtype=capi.F16,
           q_norm=ADDRESS, q_norm_pitch=0, k_norm=ADDRESS, k_norm_pitch=0, norm_dtype=capi.F16, eps=1e-6):
    return ttmi.ttmi_rotary_append_normed(P(qkv), qkv_pitch, P(q), q_pitch, heads, ctypes.byref(c) if c else None, ctypes.byref(b) if b else None, P(inv_freq), rotary,
                                          interleaved, 1.0, P(q_norm), q_norm_pitch, P(k_norm), k_norm_pitch, norm_dtype, eps, dtype, None)


def attend(ttmi, c, b, q=ADDRESS, q_pitch=256, out=2 * ADDRESS, out_pitch=256, heads=4, max_tokens=0, max_length=0, scale=0.125, window=8, sinks=4, families=ADDRESS,
           family_count=0, max_shared=0, workspace=None, bytes=0, dtype=capi.F16, sight=True):
    s = capi.PagedSight(window, sinks, families, family_count, max_shared)
    return ttmi.ttmi_paged_attention_sight(P(q), q_pitch, P(out), out_pitch, heads, ctypes.byref(c) if c else None, ctypes.byref(b) if b else None, max_tokens,
                                           max_length, scale, 1, ctypes.byref(s) if sight else None, P(workspace), bytes, dtype, None)


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


def test_append_refuses(lib):
    inf, nan = float("inf"), float("nan")
    for changes in (dict(qkv=None), dict(q=None), dict(inv_freq=None), dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(qkv_pitch=511), dict(q_pitch=255),
                    dict(q=ADDRESS), dict(qkv=ADDRESS + 1), dict(qkv=ADDRESS + 2, interleaved=1), dict(norm_dtype=capi.BF16), dict(norm_dtype=capi.I8),
                    dict(q_norm_pitch=63), dict(k_norm_pitch=-64), dict(eps=-1e-6), dict(eps=nan), dict(eps=inf), dict(q_norm=ADDRESS + 1),
                    dict(k_norm=ADDRESS + 2, norm_dtype=capi.F32), dict(q_norm=ADDRESS + 2, interleaved=1), dict(k_norm_pitch=65, interleaved=1)):
        assert append(lib, cache(), batch(), **changes) == -1, changes
    # nothing to do
    assert append(lib, cache(), batch(tokens=0)) == 0 and append(lib, cache(), batch(batch=0)) == 0


def test_attention_refuses(lib):
    for changes in (dict(q=None), dict(out=None), dict(q=ADDRESS + 8), dict(out=ADDRESS + 2), dict(q_pitch=252), dict(q_pitch=258), dict(out_pitch=260),
                    dict(window=-1), dict(sinks=-1), dict(max_tokens=-1), dict(max_length=-1), dict(family_count=-1), dict(max_shared=-1), dict(scale=0.0),
                    dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=2.3587e38), dict(sight=False)):
        for families in (ADDRESS, None):
            assert attend(lib, cache(), batch(), **{"families": families, **changes}) == -1, changes
    for d in (16, 80, 96, 256):
        assert attend(lib, cache(head_dim=d), batch(), q_pitch=4 * d, out_pitch=4 * d) == -1
    assert attend(lib, cache(), batch(tokens=0)) == 0 and attend(lib, cache(), batch(batch=0)) == 0
    assert attend(lib, cache(), batch(), families=ADDRESS + 2) == -1


def room(lib, sequences, tokens, heads=32, kv_heads=8, d=128, most=0, longest=0, window=0, sinks=0, families=ADDRESS, count=0, shared=0, dtype=capi.F16, pitch=1 << 14,
         page=16):
    n = ctypes.c_int64(-7)
    s = capi.PagedSight(window, sinks, families, count, shared)
    rc = lib.ttmi_paged_attention_sight_workspace(ctypes.byref(cache(pages=1 << 20, kv_heads=kv_heads, head_dim=d, page_size=page)),
                                                  ctypes.byref(batch(batch=sequences, tokens=tokens, table_pitch=pitch)), heads, most, longest, ctypes.byref(s), dtype,
                                                  ctypes.byref(n))
    return n.value if rc == 0 else rc


def test_workspace_refuses(lib):
    n = ctypes.c_int64(-7)
    s = capi.PagedSight(0, 0, ADDRESS, 0, 0)
    call = lambda c, b, sight, out: lib.ttmi_paged_attention_sight_workspace(c, b, 4, 0, 0, sight, capi.F16, out)
    args = [ctypes.byref(x) for x in (cache(), batch(), s, n)]
    assert call(*args) == 0
    for i in range(4):
        assert call(*[None if j == i else a for j, a in enumerate(args)]) == -1, i
    assert room(lib, 2, 3, window=-1) == -1 and room(lib, 2, 3, sinks=-1) == -1 and room(lib, 2, 3, count=-1) == -1 and room(lib, 2, 3, shared=-1) == -1
    assert room(lib, 2, 0) == 0


@pytest.mark.parametrize("dtype,heads,kv_heads,d,families,shared,faster", [
    (capi.BF16, 32, 8, 128, (4, 4), 1000, False), (capi.BF16, 32, 8, 128, (4, 8), 1000, False), (capi.BF16, 32, 8, 128, (1, 16), 1000, False), (capi.F32, 12, 12, 64, (1, 4), 1000, False),
    (capi.F16, 12, 12, 64, (8, 8), 1000, False), (capi.BF16, 32, 8, 128, (8, 2), 1000, False), (capi.BF16, 32, 8, 128, (4, 8), 2000, True), (capi.BF16, 32, 8, 128, (1, 256), 1000, True),
    (capi.BF16, 32, 8, 128, (16, 4), 2000, True), (capi.BF16, 32, 8, 128, (2, 4), 3000, True), (capi.F16, 12, 12, 64, (1, 64), 1500, True), (capi.F16, 12, 12, 64, (8, 8), 1500, True),
    (capi.F32, 12, 12, 64, (1, 4), 3000, True), (capi.F32, 12, 12, 64, (1, 64), 1000, True), (capi.F32, 32, 8, 128, (1, 64), 1500, True), (capi.F32, 32, 8, 128, (1, 64), 1000, False)])
def test_families_are_shared_where_that_was_measured_to_be_faster(lib, dtype, heads, kv_heads, d, families, shared, faster):
    """(families, sequences of each), a token and 50 keys of its own each: as the times say where the two differ, and that nothing is shared where they are level (4 families of 8
    behind 1000 keys 21.9 / 21.5 us).  What a call asks for as its workspace tells which way it goes."""
    count, members = families
    n, held = count * members, shared // 16 * 16
    asked = dict(heads=heads, kv_heads=kv_heads, d=d, most=1, longest=shared + 51, dtype=dtype, pitch=-(-(shared + 51) // 16))
    assert (room(lib, n, n, count=count, shared=held, **asked) != room(lib, n, n, families=None, **asked)) == faster
    assert room(lib, n, n, **asked) != room(lib, n, n, families=None, **asked)  # unknown: as they come


@pytest.mark.parametrize("dtype,heads,kv_heads,d,families,tokens,shared,faster", [
    (capi.BF16, 32, 8, 128, (1, 32), 20, 1000, False), (capi.BF16, 32, 8, 128, (8, 4), 20, 1000, False), (capi.BF16, 32, 8, 128, (8, 4), 50, 2000, False),
    (capi.BF16, 32, 8, 128, (1, 16), 50, 2000, False), (capi.BF16, 8, 4, 64, (4, 2), 150, 5000, False), (capi.F32, 32, 8, 128, (8, 4), 50, 700, False),
    (capi.F32, 16, 2, 128, (4, 2), 50, 2000, False), (capi.BF16, 32, 8, 128, (1, 100), 6, 4000, True), (capi.F32, 12, 12, 64, (1, 48), 20, 700, True),
    (capi.F32, 12, 12, 64, (1, 4), 50, 2000, True), (capi.BF16, 32, 8, 128, (1, 16), 100, 20000, True)])
def test_families_with_chunks_are_shared_where_that_was_measured_to_be_faster(lib, dtype, heads, kv_heads, d, families, tokens, shared, faster):
    """The same of sequences with several new tokens each, where either way took up to twice as long as the other."""
    count, members = families
    n, held = count * members, shared // 16 * 16
    longest = shared + 50 + tokens
    asked = dict(heads=heads, kv_heads=kv_heads, d=d, most=tokens, longest=longest, dtype=dtype, pitch=-(-longest // 16))
    assert (room(lib, n, n * tokens, count=count, shared=held, **asked) != room(lib, n, n * tokens, families=None, **asked)) == faster


@pytest.mark.parametrize("dtype,heads,kv_heads,d,families,tokens,shared,window,sinks,faster", [
    (capi.BF16, 32, 8, 128, (16, 4), 1, 8000, 1500, 4, False), (capi.BF16, 12, 12, 64, (8, 4), 1, 8000, 1500, 4, False), (capi.F32, 32, 8, 128, (16, 4), 1, 8000, 500, 4, False),
    (capi.F32, 32, 8, 128, (1, 16), 1, 8000, 500, 4, False), (capi.F32, 32, 8, 128, (8, 4), 20, 2000, 1500, 4, False), (capi.BF16, 32, 8, 128, (8, 4), 20, 8000, 4000, 4, False),
    (capi.BF16, 32, 8, 128, (1, 64), 1, 8000, 4000, 4, True), (capi.BF16, 32, 8, 128, (1, 64), 1, 8000, 1500, 9000, True), (capi.F32, 32, 8, 128, (1, 64), 1, 8000, 4000, 4, True)])
def test_families_behind_windows_are_shared_where_that_was_measured_to_be_faster(lib, dtype, heads, kv_heads, d, families, tokens, shared, window, sinks, faster):
    """Common keys that a window hides cost those who share them some of what they would if they were seen, and the others nothing."""
    count, members = families
    n, held = count * members, shared // 16 * 16
    longest = shared + 50 + tokens
    asked = dict(heads=heads, kv_heads=kv_heads, d=d, most=tokens, longest=longest, dtype=dtype, pitch=-(-longest // 16), window=window, sinks=sinks)
    assert (room(lib, n, n * tokens, count=count, shared=held, **asked) != room(lib, n, n * tokens, families=None, **asked)) == faster


@pytest.mark.parametrize("dtype", [capi.F32, capi.F16])
def test_workspace_does_not_grow_with_keys_that_a_window_hides(lib, dtype):
    """300 tokens that see their last 500 keys and the first 20: as much room with a table for 2^24 positions as with one for 2^12, and with the largest numbers as with
    those that hide nothing."""
    sizes = [room(lib, 1, 300, 4, 2, 64, 300, 0, 500, 20, None, dtype=dtype, pitch=pitch) for pitch in (1 << 8, 1 << 20)]
    assert sizes[0] == sizes[1] and 0 < sizes[0] <= 300 * 4 * 66 * 4 * 20
    for tokens in (1, 300):
        sizes = [room(lib, 1, tokens, 4, 2, 64, tokens, 0, window, sinks, None, dtype=dtype, pitch=1 << 12)
                 for window in (1 << 22, 1 << 30, (1 << 31) + 5, (1 << 63) - 1 - tokens, (1 << 63) - 1) for sinks in (7, 1 << 20, (1 << 63) - 1)]
        assert min(sizes) >= 0 and max(sizes) < 1 << 30


def test_launches_that_are_too_large_are_refused(lib):
    assert attend(lib, cache(kv_heads=1), batch(tokens=1 << 20), heads=1 << 10, q_pitch=1 << 16, out_pitch=1 << 16) == -1
    assert attend(lib, cache(), batch(batch=1 << 22)) == -1
    assert b"than one launch takes" in lib.ttmi_last_error()
    # rows that the sequences' own keys and the families' fill a launch with between them
    assert attend(lib, cache(kv_heads=128), batch(batch=4, tokens=(1 << 23) - 1), heads=128, q_pitch=1 << 13, out_pitch=1 << 13) == -1
    assert b"than one launch takes" in lib.ttmi_last_error()


def test_python_calls_that_are_refused():
    kv = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    ints = [torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)]
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.float16)
    norm = torch.ones(64)
    for call in (lambda: tt.paged_attention(q, kv, kv.clone(), *ints, window=3, sinks=1), lambda: tt.rotary_append(qkv, kv, kv.clone(), *ints, q_norm=norm),
                 lambda: tt.paged_attention(q, kv, kv.clone(), *ints, families=torch.zeros(1, 3, dtype=torch.int32))):
        with pytest.raises(tt.cxx.EnforceNotMet, match="not on the GPU"):
            call()
    for call in (lambda: tt.paged_attention(q, kv, kv.clone(), *ints, families=3), lambda: tt.rotary_append(qkv, kv, kv.clone(), *ints, k_norm=[1.0])):
        with pytest.raises(tt.cxx.EnforceNotMet, match="expected a tensor"):
            call()


def test_families_are_taken_where_they_save_reads(lib):
    """One token each of 8 or 64 sequences, 32 and 8 heads of 128 in fp16 (4 KB a key): common keys are read once, which needs room for partial results, where that is much or not known."""
    alone = [room(lib, n, n, most=1, longest=longest, families=None) for n, longest in ((8, 600), (64, 600))]
    assert alone == [0, 0]  # (short contexts are not cut)
    call = lambda n, shared, count=1: room(lib, n, n, most=1, longest=600, count=count, shared=shared)
    assert call(8, 512) == call(64, 64) == call(64, 256) == call(64, 512, 60) == 0
    assert call(64, 4096) > 0 and call(8, 16384) > 0 and call(8, 0) > 0 and call(8, 512, 0) > 0
