"""A paged key-value cache for attention over all previous tokens, and one new token's attention to it.

The one full-attention layer of the reference's models (train/train_2048_condM_layer_ablation.py:214-286) needs every
key and value of a sequence.  Pages of a fixed number of positions let sequences of different lengths share one block of memory
and grow without copies; in 8 bits (e4m3 with a power-of-two scale per row) the cache takes half of what bf16 takes.  The
reference has no counterpart: its generate() re-runs the prefix (train/train_2048_condU.py:463-487).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib


def paged_kv_write(k, v, kv_pages, block_table, cu_seqlens, start=None, kv_scale=None):
    """The keys and values of a ragged batch into their pages.

    k, v [tokens,H,D] bf16 or fp32 (token and head strides may be any multiple of 8 elements, e.g. slices of a fused projection's output);
    kv_pages [P,H,page,2,D] bf16, fp32 or float8_e4m3fn (then kv_scale [P,H,page,2] float8_e8m0fnu), updated in place; block_table int32
    [S,columns]: the page of positions [c*page, (c+1)*page) of a sequence; cu_seqlens int32 [S+1]: token t belongs to the sequence s with
    cu_seqlens[s] <= t < cu_seqlens[s+1] and goes to position start[s] + t - cu_seqlens[s] (start int32 [S], default 0).  Tokens of no sequence,
    and positions for which the table names no page of the cache, are left out."""
    _lib.native().paged_kv_write(k, v, kv_pages, block_table, cu_seqlens, start, kv_scale)


def paged_kv_read(kv_pages, block_table, cu_seqlens, tokens: int, start=None, kv_scale=None, dtype=torch.bfloat16):
    """(k, v) [tokens,H,D] of a ragged batch of positions, the inverse of paged_kv_write: rows of no sequence are zeros, positions without a
    page are NaN."""
    return _lib.native().paged_kv_read(kv_pages, block_table, cu_seqlens, tokens, start, kv_scale, dtype)


def paged_attention_step(q, k_new, v_new, kv_pages, block_table, lengths, kv_scale=None, scale=None, max_length=None, out=None):
    """Attention of one new token per sequence: q [S,Hq,D] bf16 or fp32, Hq a multiple of the cache's H (query head i reads key-value head
    i // (Hq / H)) -> [S,Hq,D].

    lengths int32 [S] on the device counts the new token: k_new, v_new [S,H,D] are stored at position lengths[s] - 1 and attended to as stored
    (None, None: nothing is stored, all lengths[s] positions are read).  Sequences may share pages that no token is stored in.  A length of 0
    gives zeros and stores nothing.  max_length: no length is above it (default: what the table has room for); a longer one gives NaN, and so
    does a position for which the table names no page.  The cache's length is split over the GPU by max_length, so a tight bound is faster for
    few sequences.  scale: of the scores, positive in fp32, default 1/sqrt(D).

    Sums are held in fp32; on tensor cores a probability enters the product with the values as two 16-bit numbers, off by 2^-15 of it over bf16
    pages and by 2^-22 over 8-bit pages (2^-33 of the largest term where it is that small).  Fastest with bf16 queries over bf16 or 8-bit pages
    of a multiple of 16 positions, D a multiple of 32, 48 or 80."""
    return _lib.native().paged_attention_step(q, k_new, v_new, kv_pages, block_table, lengths, kv_scale, scale, max_length, out)


class PagedKVCache:
    """Pages for the keys and values of L layers and S sequences, one block table and one length per sequence for all layers.

    kv [L,P,H,page,2,D] (`dtype` bf16, fp32 or float8_e4m3fn; then kv_scale [L,P,H,page,2] float8_e8m0fnu), block_table int32 [S,columns] and
    lengths int32 [S] are device tensors that never move, so a captured step replays on the lengths and pages of the day.  Which page
    belongs to whom is kept on the host; `extend`, `advance`, `reserve` and `release` are host calls, made outside a capture."""

    def __init__(self, layers, sequences, heads, head_dim, max_length, pages=None, page_size=64, dtype=torch.bfloat16, device="cuda"):
        if min(layers, sequences, heads, page_size, max_length) < 1:
            raise ValueError("paged cache: layers, sequences, heads, page_size and max_length must be positive")
        if dtype not in (torch.bfloat16, torch.float32, torch.float8_e4m3fn):
            raise TypeError(f"paged cache: dtype must be bfloat16, float32 or float8_e4m3fn, got {dtype}")
        self.page_size, self.max_length = page_size, max_length
        columns = -(-max_length // page_size)
        pages = sequences * columns if pages is None else pages
        if pages < 1:
            raise ValueError("paged cache: pages must be positive")
        e4m3 = dtype is torch.float8_e4m3fn
        shape = (layers, pages, heads, page_size, 2)
        self.kv = torch.zeros(*shape, head_dim, dtype=torch.uint8 if e4m3 else dtype, device=device).view(dtype)
        self.kv_scale = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu) if e4m3 else None
        self.block_table = torch.full((sequences, columns), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._table = torch.full((sequences, columns), -1, dtype=torch.int32)
        self._owned = [[] for _ in range(sequences)]
        self._length = [0] * sequences
        self._free = list(range(pages - 1, -1, -1))

    @property
    def step_dtype(self):
        """The type of q, k and v that `step` takes for what the cache holds (8-bit caches: bf16; fp32 works too)."""
        return torch.bfloat16 if self.kv_scale is not None else self.kv.dtype

    def _scale(self, layer):
        return None if self.kv_scale is None else self.kv_scale[layer]

    def reserve(self, sequence, length):
        """Pages for `length` positions of a sequence.  Raises RuntimeError, and changes nothing, when there are not enough."""
        self._reserve({sequence: length})

    def _reserve(self, wanted):
        more = {}
        for s, n in wanted.items():
            if n > self.max_length:
                raise ValueError(f"paged cache: {n} positions, but max_length is {self.max_length}")
            more[s] = max(0, -(-n // self.page_size) - len(self._owned[s]))
        if sum(more.values()) > len(self._free):
            raise RuntimeError(f"paged cache: out of pages ({sum(more.values())} wanted, {len(self._free)} free)")
        for s, n in more.items():
            for _ in range(n):
                page = self._free.pop()
                self._table[s, len(self._owned[s])] = page
                self._owned[s].append(page)
        if any(more.values()):
            self.block_table.copy_(self._table)

    def release(self, sequence):
        """Gives a sequence's pages back; its slot of the batch is empty (length 0) until the next `extend`."""
        self._free.extend(reversed(self._owned[sequence]))
        self._owned[sequence] = []
        self._table[sequence] = -1
        self._length[sequence] = 0
        self.block_table.copy_(self._table)
        self.lengths[sequence] = 0

    def extend(self, counts: Sequence[int]):
        """Room for counts[s] more positions of every sequence; call it once per chunk of a prompt, before the layers `write` it.  Returns what `write` and
        `read` take: (cu_seqlens, start) on the device and the number of tokens."""
        counts = [int(c) for c in counts]
        if len(counts) != len(self._length) or min(counts) < 0:
            raise ValueError("paged cache: one count per sequence, none negative")
        self._reserve({s: self._length[s] + c for s, c in enumerate(counts)})
        start, cu = list(self._length), [0]
        for s, c in enumerate(counts):
            cu.append(cu[-1] + c)
            self._length[s] += c
        to = lambda x: torch.tensor(x, dtype=torch.int32, device=self.kv.device)  # noqa: E731
        self.lengths.copy_(to(self._length))
        return to(cu), to(start), cu[-1]

    def write(self, layer, k, v, chunk):
        """k, v [tokens,H,D] of a chunk that `extend` made room for."""
        paged_kv_write(k, v, self.kv[layer], self.block_table, chunk[0], chunk[1], self._scale(layer))

    def read(self, layer, dtype=torch.bfloat16):
        """(k, v, cu_seqlens): every position of every sequence, [tokens,H,D] in sequence order."""
        cu = torch.tensor([0] + list(self._length), dtype=torch.int64).cumsum(0)
        dev = cu.to(torch.int32).to(self.kv.device)
        k, v = paged_kv_read(self.kv[layer], self.block_table, dev, int(cu[-1]), None, self._scale(layer), dtype)
        return k, v, dev

    def advance(self):
        """Room for one more token of every sequence that has any; call it once per token before the layers run."""
        live = [s for s, n in enumerate(self._length) if n]
        self._reserve({s: self._length[s] + 1 for s in live})
        for s in live:
            self._length[s] += 1
        # on the device, so that the host does not wait for the steps in flight
        self.lengths.add_(1 if len(live) == len(self._length) else self.lengths > 0)

    def step(self, layer, q, k_new, v_new, scale=None, max_length: Optional[int] = None, out=None):
        """One new token per sequence against layer `layer` (see paged_attention_step); max_length defaults to the longest sequence, rounded up to whole
        pages.  A captured step keeps the bound it was captured with: give one that covers the replays."""
        if max_length is None:
            max_length = -(-max(self._length) // self.page_size) * self.page_size
        return paged_attention_step(q, k_new, v_new, self.kv[layer], self.block_table, self.lengths, self._scale(layer), scale, max_length, out)
