"""A decoder's keys and values in pages, and the operators over them.

A cache of one layer is two dense tensors, keys and values [pages, kv_heads, page_size, head_dim].  A sequence's token i lies in slot
i % page_size of the i // page_size-th of its pages; pages lie anywhere, and sequences may share them.  A batch is given by three int32 tensors
on the GPU: `table` [batch, n] (the pages of each sequence in order; what stands behind its last page is not read), `starts` [batch + 1] (the new
tokens of sequence b are rows starts[b] to starts[b + 1] of the packed tensors: none, one or many) and `lengths` [batch] (its keys, the new
tokens' among them).  Rows behind starts[batch] are neither read nor written.

The functions are enqueued on torch's current stream and share nothing between calls; they can be recorded into a graph after one call outside, and
replayed with other contents of all tensors.  A page outside the cache, or a token that the table has no page for, is reported by the next
`cxx.synchronize()`.  No counterpart in the reference, whose layer cache is a dense tensor that every step copies (modules.py:60-103).
"""
import math
from typing import Optional, Sequence

import torch

from .. import cxx

__all__ = ['PagedCache', 'PagedBatch', 'rotary_append', 'paged_attention', 'copy_pages', 'rotary_frequencies']

_LEAST_SHARED = 128  # keys that the kernels take as shared: the step of their work

_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)  # absent from builds without a device
_current_device, _is_initialized = torch.cuda.current_device, torch.cuda.is_initialized


def _here():
    """The current device and stream; -1 where there is none (the operators then say what is wrong with their tensors)."""
    if _raw_stream is None or not _is_initialized():
        return -1, 0
    device = _current_device()
    return device, _raw_stream(device)


def _empty_bytes(n):
    return torch.empty(n, dtype=torch.uint8, device='cuda')


def rotary_append(qkv: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                  lengths: torch.Tensor, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                  amplitude: float = 1.0, out: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                  k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Turns the new tokens' queries and keys by their positions and stores keys and values into their pages.

    qkv: [tokens, (heads + 2 kv_heads) * head_dim] or [tokens, heads + 2 kv_heads, head_dim], queries first; rows may lie any distance apart.
    inv_freq: float64 on the GPU; pair i of the first 2 * len(inv_freq) elements of a head turns by position * inv_freq[i] (`rotary_frequencies`
    makes them), None: nothing turns.  interleaved: pairs are neighbours (2i, 2i + 1), else (i, i + len(inv_freq)).
    q_norm, k_norm: where given, queries / keys are normed head by head before they turn, x / sqrt(mean(x^2) + eps) * weight: float32 or qkv's type, [head_dim] for
    all heads or [heads, head_dim] / [kv_heads, head_dim].  Everything is computed in 32 bits (a head's sum of squares has to stay below 2^128) and rounded once.
    -> the queries [tokens, heads, head_dim]: `out` if given, which may be the queries' part of qkv itself."""
    if out is None:
        shape = qkv.shape
        _, kv_heads, _, d = keys.shape
        heads = (shape[1] // d if len(shape) == 2 else shape[1]) - 2 * kv_heads
        if heads < 1:
            raise ValueError("qkv has no room for queries beside the cache's heads")
        out = qkv.new_empty((shape[0], heads, d))
    if q_norm is None and k_norm is None:
        cxx.rotary_append(qkv, keys, values, table, starts, lengths, inv_freq, interleaved, amplitude, out, *_here())
    else:
        cxx.rotary_append(qkv, keys, values, table, starts, lengths, inv_freq, interleaved, amplitude, out, *_here(), q_norm, k_norm, eps)
    return out


def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                    lengths: torch.Tensor, max_tokens: int = 0, max_length: int = 0, scale: Optional[float] = None, causal: bool = True,
                    window: int = 0, out: Optional[torch.Tensor] = None, sinks: int = 0, families: Optional[torch.Tensor] = None,
                    family_count: int = 0, max_shared: int = 0) -> torch.Tensor:
    """softmax(scale * q k^T) v of the new tokens over their sequences' keys: up to a token's own position if causal, all of them otherwise;
    window > 0: only the last `window` up to its own, and with sinks > 0 the first `sinks` of its sequence besides.  A token that sees no key gets zeros; where it sees some, all with a score of minus
    infinity, NaN, as zero divided by zero is.  Sums and statistics are held in 32 bits; in 16-bit types the probabilities are rounded to the type for
    their product with v (and divided by the sum of the rounded ones).  The sum of |v| over a token's keys has to stay below 2^120.

    q: [tokens, heads * head_dim] or [tokens, heads, head_dim], head_dim 64 or 128; rows may lie any multiple of 16 bytes apart.  heads is a
    multiple of kv_heads: query head h reads key/value head h // (heads // kv_heads).  scale: positive, 1 / sqrt(head_dim) by default.
    max_tokens, max_length: the most new tokens and keys of a sequence, where known: they choose how the work is cut, not what is computed.
    families: int32 [batch, 3] on the GPU: neighbouring sequences whose first keys lie in the same pages may be a family, whose common keys are read once for all of them.
    The row of each of its sequences is (number of the first of them, number behind the last, keys they have in common); of one that is on its own (its own number, the next,
    0); one whose row is not that of the first it names is on its own as well.  The common keys are read where the first one's row of the table says, in steps of 128 (fewer are not
    shared).  The result is that without families but for roundings.
    family_count, max_shared: how many families there are and the most keys of one, where known: hints as well.  `PagedCache.extend(..., share=True)` fills in all three.
    -> like q: `out` if given."""
    if out is None:
        out = torch.empty_like(q)
    if sinks == 0 and families is None:
        cxx.paged_attention(q, keys, values, table, starts, lengths, out, max_tokens, max_length, scale, causal, window, _empty_bytes, *_here())
    else:
        cxx.paged_attention(q, keys, values, table, starts, lengths, out, max_tokens, max_length, scale, causal, window, _empty_bytes, *_here(), sinks, families,
                            family_count, max_shared)
    return out


def copy_pages(keys: torch.Tensor, values: torch.Tensor, sources: Sequence[int], destinations: Sequence[int]) -> None:
    """Page destinations[i] becomes a copy of page sources[i], in keys and values [pages, kv_heads, page_size, head_dim] or, of all layers,
    [layers, pages, kv_heads, page_size, head_dim].  A page must not be a destination twice, nor a source and a destination."""
    cxx.copy_pages(keys, values, sources, destinations, *_here())


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, stretch: float = 1.0, trained_length: Optional[int] = None,
                       slow_turns: float = 1.0, fast_turns: float = 32.0, device=None) -> torch.Tensor:
    """inv_freq for `rotary_append`, float64 [rotary_dim / 2]: base^(-2i / rotary_dim).

    stretch > 1 serves contexts `stretch` times as long as the model was trained for: all positions are divided by it.  With `trained_length` only
    those pairs are that would not have come round in training: pairs that made at most `slow_turns` turns over trained_length tokens are divided
    by stretch, pairs that made at least `fast_turns` are left, those between are blended linearly in their number of turns."""
    if rotary_dim % 2 or rotary_dim < 0:
        raise ValueError("rotary_dim must be even")
    if stretch <= 0 or base <= 0:
        raise ValueError("base and stretch must be positive")
    inv_freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1))
    if trained_length is None:
        inv_freq = inv_freq / stretch
    else:
        if not slow_turns < fast_turns:
            raise ValueError("slow_turns must be less than fast_turns")
        turns = trained_length * inv_freq / (2 * math.pi)
        kept = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        inv_freq = inv_freq * kept + inv_freq / stretch * (1 - kept)
    return inv_freq.to(device if device is not None else 'cuda')


class PagedBatch:
    """The sequences of one step as the operators take them; all layers of the step share it."""

    def __init__(self, table: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, max_tokens: int = 0, max_length: int = 0,
                 families: Optional[torch.Tensor] = None, family_count: int = 0, max_shared: int = 0):
        self.table, self.starts, self.lengths, self.max_tokens, self.max_length = table, starts, lengths, max_tokens, max_length
        self.families, self.family_count, self.max_shared = families, family_count, max_shared


class PagedCache:
    """Keys and values of all layers of a decoder in pages, and the book of who holds which page.

        cache = PagedCache(layers, kv_heads, head_dim, pages, page_size, dtype)
        a = cache.add()                                   # an empty sequence
        step = cache.extend([a], [len(prompt)])           # room for its tokens
        for layer in ...:
            q = cache.append(layer, qkv, step, inv_freq)  # keys and values of the new tokens
            context = cache.attend(layer, q, step)
        b = cache.fork(a)                                 # shares a's pages; a page that both would write is copied by extend()
        cache.free(a)

    `attend` reads heads of 64 or 128; the rest takes any multiple of 16 up to 256.  `pool` is the book itself (cxx.PagePool).  Pages that are freed may be handed out by the next `extend`; work of earlier steps that still reads
    them has to be on the same stream."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_size: int = 16, dtype: torch.dtype = torch.float16, device=None):
        self.pool = cxx.PagePool(pages, page_size)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.keys = torch.zeros(shape, dtype=dtype, device=device if device is not None else 'cuda')
        self.values = torch.zeros_like(self.keys)

    def add(self) -> int:
        return self.pool.add()

    def fork(self, sequence: int) -> int:
        """A sequence with the same tokens, which lie in the same pages until one of the two grows."""
        return self.pool.fork(sequence)

    def free(self, sequence: int) -> None:
        self.pool.free(sequence)

    def truncate(self, sequence: int, length: int) -> None:
        """Back to the first `length` tokens (as after speculated tokens that were refused)."""
        self.pool.truncate(sequence, length)

    def length(self, sequence: int) -> int:
        return self.pool.length(sequence)

    def _move(self, pairs):
        if pairs:
            copy_pages(self.keys, self.values, [p[0] for p in pairs], [p[1] for p in pairs])

    def extend(self, sequences: Sequence[int], tokens: Sequence[int], share: bool = False) -> PagedBatch:
        """Room for tokens[i] new tokens of sequences[i], and the batch of that step.  Shared pages that would be written are copied first.
        share: neighbours in `sequences` that begin with the same 128 or more tokens in the same pages (forks of one another) are a family in this step, and `attend`
        reads those keys once for all of them.
        A call that raises, for want of free pages or because a copy or the batch cannot be made, leaves every sequence with the tokens it had."""
        self._move(self.pool.copies_of(sequences, tokens))  # (to free pages: the book follows when they have been enqueued)
        before = [self.pool.length(s) for s in sequences]
        self.pool.extend(sequences, tokens)
        try:
            return self._batch(sequences, tokens, [n + more for n, more in zip(before, tokens)], before if share else None)
        except BaseException:
            for s, n in zip(sequences, before):
                self.pool.truncate(s, n)
            raise

    def _batch(self, sequences, tokens, lengths, before):
        longest = max(lengths, default=0)
        starts = [0]
        for n in tokens:
            starts.append(starts[-1] + n)
        table = self.pool.table(sequences, max(1, -(-longest // self.pool.page_size)))
        rows, family_count, max_shared = self.pool.families(sequences, before, _LEAST_SHARED) if before is not None else (None, 0, 0)
        # one copy to the device: [table | starts | lengths | families]
        parts = [torch.from_numpy(table).flatten(), torch.tensor(starts + lengths, dtype=torch.int32)]
        if family_count:
            parts.append(torch.from_numpy(rows).flatten())
        packed = torch.cat(parts)
        if self.keys.is_cuda:
            packed = packed.pin_memory().to(self.keys.device, non_blocking=True)
        n, width = table.shape
        at = n * width + n + 1
        return PagedBatch(packed[:n * width].view(n, width), packed[n * width:at], packed[at:at + n], max(tokens, default=0), longest,
                          packed[at + n:].view(n, 3) if family_count else None, family_count, max_shared)

    def compact(self) -> int:
        """Moves live pages to the lowest numbers -> how many moved.  Batches made before are void.  A call that raises has changed nothing."""
        moves = self.pool.moves_of()
        self._move(moves)  # (to free pages, as above)
        self.pool.compact()
        return len(moves)

    def append(self, layer: int, qkv: torch.Tensor, batch: PagedBatch, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
               amplitude: float = 1.0, out: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
        """`rotary_append` into this cache."""
        return rotary_append(qkv, self.keys[layer], self.values[layer], batch.table, batch.starts, batch.lengths, inv_freq, interleaved, amplitude, out,
                             q_norm, k_norm, eps)

    def attend(self, layer: int, q: torch.Tensor, batch: PagedBatch, scale: Optional[float] = None, causal: bool = True, window: int = 0,
               out: Optional[torch.Tensor] = None, sinks: int = 0) -> torch.Tensor:
        """`paged_attention` over this cache, with the families of a batch made with `share`."""
        return paged_attention(q, self.keys[layer], self.values[layer], batch.table, batch.starts, batch.lengths, batch.max_tokens, batch.max_length,
                               scale, causal, window, out, sinks, batch.families, batch.family_count, batch.max_shared)
