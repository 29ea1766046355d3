"""A cache for streams that never end, kept on the device.

`Cache` (cache.py) keeps lengths and page lists on the host, which sends a step's tables along with its tokens.  Here they live on
the device: a step names its sequences and how many rows each brings, and the kernels of csrc/stream_tables.cu lay out its
rows, page tables and slot map, take pages off a stack and give back those that left the window.  A decode step
therefore replays as a graph for as long as its streams go on, without the host: its sequences advance by themselves.

A sequence keeps its last `window` positions and its first `first` ones (0: all of them); memory per stream is bounded by
ceil(first / page) + ceil(window / page) + 1 pages and what a step brings.  Positions go on being counted, so a stream may
be as long as its page list (`max_len`).

    cache = StreamCache(layers, kv_heads, head_dim, max_seqs=64, max_tokens=1 << 20, max_len=1 << 20, window=4096, first=4, device="cuda")
    slots = [cache.open() for _ in requests]
    step = cache.plan(len(slots), rows, max_qlen)       # buffers of a step of this shape: keep it, its addresses stay
    step.set(slots, row_counts)
    cache.begin(step)                                   # tables; the sequences are longer
    cache.store(layer, step, k, v)                      # per layer
    cache.attend(layer, step, out, q, heads)
    cache.check()                                       # raises if a step since the last check was refused (waits: not in every step)
    cache.close(slots)
"""
from __future__ import annotations

import math
from typing import Sequence

import torch

from ..ops import kernels
from .allocator import CacheError, CacheFull, IdPool
from .cache import PAGE_SIZE


class StreamStep:
    """The device buffers of a step of `n_seqs` sequences and `n_rows` rows, named as the kernels of a step know them."""

    def __init__(self, n_seqs: int, n_rows: int, max_qlen: int, max_kvlen: int, width: int, device):
        words = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)
        self.n_seqs, self.n_rows, self.max_qlen, self.max_kvlen = n_seqs, n_rows, max_qlen, max_kvlen
        self.slots, self.row_counts = words(n_seqs), words(n_seqs)           # what the step asks for
        self.slots.fill_(-1)
        self.seq_slot, self.seq_qlen = words(n_seqs), words(n_seqs)          # what it got
        self.seq_pos0, self.seq_qstart = words(n_seqs), words(n_seqs)
        self.row_seq, self.row_pos, self.slot_map = words(n_rows), words(n_rows), words(n_rows)
        self.table = words(n_seqs, width)

    def set(self, slots: Sequence[int], row_counts: Sequence[int]) -> None:
        """The step's sequences (slot -1: padding, whose rows touch no cache) and how many rows each brings."""
        slots, row_counts = [int(s) for s in slots], [int(n) for n in row_counts]
        live = [s for s in slots if s >= 0]
        if len(slots) != self.n_seqs or len(row_counts) != self.n_seqs or sum(row_counts) != self.n_rows:
            raise CacheError(f"a step of {self.n_seqs} sequences and {self.n_rows} rows, got {len(slots)} and {sum(row_counts)}")
        if len(set(live)) != len(live):
            raise CacheError("a sequence is named twice in a step")
        if row_counts and (min(row_counts) < 0 or max(row_counts) > self.max_qlen):
            raise CacheError(f"sequences of {min(row_counts)} to {max(row_counts)} rows in a step of at most {self.max_qlen} each")
        self.slots.copy_(torch.tensor(slots, dtype=torch.int32))
        self.row_counts.copy_(torch.tensor(row_counts, dtype=torch.int32))


class StreamCache:
    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, *, max_seqs: int, max_tokens: int, max_len: int, device,
                 window: int = 0, first: int = 0, v_head_dim: int | None = None, page_size: int = PAGE_SIZE,
                 dtype: torch.dtype = torch.bfloat16):
        """`max_tokens`: positions all sequences may hold together, each rounded up to whole pages; `max_len`: the most
        positions a sequence may ever count."""
        if page_size <= 0 or page_size % 32 != 0:
            raise ValueError("page size must be a multiple of 32")
        if min(n_layers, n_kv_heads, head_dim, max_seqs, max_tokens, max_len) < 1 or window < 0 or first < 0:
            raise ValueError("sizes of a stream cache must be positive, window and first positions not negative")
        if max_len > 2 ** 31 - 2 ** 16:
            raise ValueError(f"a sequence of {max_len} positions: they are counted in 32 bits")
        window, first = (min(int(n), int(max_len)) for n in (window, first))      # (more are as many)
        self.page_size, self.window, self.first = int(page_size), int(window), int(first)
        self.nkv, self.hd, self.vd = int(n_kv_heads), int(head_dim), int(v_head_dim or head_dim)
        self.max_len = int(max_len)
        self.device, self.dtype = torch.device(device), dtype
        n_pages, width = -(-int(max_tokens) // page_size), -(-self.max_len // page_size)
        self.k = torch.zeros((n_layers, n_pages, self.nkv, page_size, self.hd), dtype=dtype, device=device)
        self.v = torch.zeros((n_layers, n_pages, self.nkv, self.vd, page_size), dtype=dtype, device=device)
        # all bookkeeping in one buffer: saved and put back by one copy
        sizes = (max_seqs, max_seqs, max_seqs * width, n_pages, 2, 2)
        at = [0]
        for n in sizes:
            at.append(at[-1] + -(-n // 4) * 4)
        self.state = torch.zeros(at[-1], dtype=torch.int32, device=device)
        self.lens, self.kept, pages, self.free, self.counts, self.refused = (self.state[o:o + n] for o, n in zip(at, sizes))
        self.pages = pages.view(max_seqs, width)
        self.pages.fill_(-1)
        self.kept.fill_(-(-self.first // page_size))
        self.free.copy_(torch.arange(n_pages - 1, -1, -1, dtype=torch.int32))     # page 0 is given out first
        self.counts.copy_(torch.tensor([n_pages, 0], dtype=torch.int32))
        self.slots = IdPool(max_seqs, "stream slot")

    # ---- sequences -----------------------------------------------------------------------
    def open(self) -> int:
        return self.slots.alloc()

    def close(self, slots: Sequence[int]) -> None:
        slots = [int(s) for s in slots]
        if len(set(slots)) != len(slots) or not all(self.slots.holds(s) for s in slots):
            raise CacheError(f"slots {slots}: not held, or named twice")
        if not slots:
            return
        words = torch.tensor(slots, dtype=torch.int32).to(self.device)
        kernels.stream_release(words, self.lens, self.kept, self.pages, self.free, self.counts, self.page_size, self.first)
        for s in slots:
            self.slots.free(s)

    # ---- a step --------------------------------------------------------------------------
    def plan(self, n_seqs: int, n_rows: int, max_qlen: int, max_kvlen: int | None = None) -> StreamStep:
        """Buffers of a step; `max_kvlen`: the most positions a sequence of it holds afterwards (None: as many as may ever be)."""
        most = self.max_len if max_kvlen is None else min(int(max_kvlen), self.max_len)
        return StreamStep(int(n_seqs), int(n_rows), int(max_qlen), most, -(-most // self.page_size), self.device)

    def begin(self, step: StreamStep) -> None:
        """Lays the step out and lets its sequences grow by its rows; a step that does not fit becomes padding (see `check`): nothing is
        stored for it, and `attend` gives zeros."""
        kernels.stream_tables(step.table, step.slot_map, step.row_seq, step.row_pos, step.seq_slot, step.seq_qlen, step.seq_pos0,
                              step.seq_qstart, step.slots, step.row_counts, self.lens, self.pages, self.free, self.counts, self.page_size,
                              keep_rows=True, refused=self.refused)
        kernels.stream_advance(step.seq_slot, step.seq_qlen, self.lens, self.kept, self.pages, self.free, self.counts, self.page_size,
                               self.window, self.first)

    def store(self, layer: int, step: StreamStep, k: torch.Tensor, v: torch.Tensor) -> None:
        kernels.store_rows(self.k[layer], self.v[layer], k, v, step.slot_map)

    def attend(self, layer: int, step: StreamStep, out: torch.Tensor, q: torch.Tensor, n_heads: int, scale: float | None = None,
               scratch: torch.Tensor | None = None, **options) -> None:
        """out [rows, heads * value width] = attention of q [rows, heads * width] over what the step's rows see.  `scratch`: float32,
        `scratch_floats(step, heads)` of them (allocated where left out).  Options as `kernels.attention` has them."""
        n = self._splits(step, n_heads)
        if n > 1 and scratch is None:
            scratch = torch.empty(self.scratch_floats(step, n_heads), dtype=torch.float32, device=self.device)
        kernels.attention(out, q, self.k[layer], self.v[layer], step.table, step, n_heads, self.nkv, self.hd, self.page_size, self.window,
                          1.0 / math.sqrt(self.hd) if scale is None else scale, n_splits=n, scratch=scratch, vd=self.vd,
                          first=self.first, **options)

    def _splits(self, step: StreamStep, n_heads: int) -> int:
        return kernels.attention_splits(step, self.nkv, n_heads // self.nkv, hd=self.hd, window=self.window, first=self.first,
                                        general=self.dtype == torch.float32 or self.vd != self.hd)

    def scratch_floats(self, step: StreamStep, n_heads: int) -> int:
        return step.n_rows * n_heads * self._splits(step, n_heads) * (max(self.hd, self.vd) + 2)

    def check(self) -> None:
        """Raises why the first step since the last call was refused, where one was.  Waits for the stream."""
        n, status = self.refused.tolist()
        if n == 0:
            return
        self.refused.zero_()
        more = f" ({n} steps were refused)" if n > 1 else ""
        if status > 0:
            raise CacheFull(f"the step needs {status} more cache pages of {self.page_size} positions than are free{more}")
        if status == -1:
            raise CacheError(f"a sequence grew longer than the step's tables (the cache takes {self.max_len} positions a sequence){more}")
        raise CacheError(("the step's rows are not those of its sequences" if status == -2 else "the step names a slot or a row count that cannot be")
                         + more)

    def lengths(self, slots: Sequence[int]) -> list[int]:
        held = self.lens.tolist()
        return [held[s] for s in slots]
