"""A paged key/value cache: what follows the ring once a prompt is done.

    cache = PagedKVCache(layers=32, num_pages=4096, heads_kv=8, head_dim=128)
    seq = cache.new_sequence()
    step = cache.step([seq], [prompt_len])          # pages, table and borders of this call
    for layer in range(32):
        q = step.append(layer, k, v, rotary=rotary, q=q)   # K rotated into the pages
        out = step.attend(layer, q)                         # causal among the new tokens
    step.commit()

    # drafted trees: parents[i] is token i's parent within its own tree, -1 the root
    step = cache.step(seqs, [len(p) for p in parents])
    mask, depth = step.tree(parents)
    ...step.append(layer, k, v, rotary=rotary, q=q, positions=step.positions(depth))
    ...step.attend(layer, q, mask=mask)
    step.accept(paths)                              # the verified path of each tree stays

    best = cache.fork(seq)                          # shares pages until one side writes
    cache.free(seq)
    cache.defragment()                              # pages in use move to the pool's front

The bookkeeping (`PageTable`) is on the host: free pages, how many sequences hold
each, and the pages of each sequence.  A fork copies nothing; before a step
writes into a page that another sequence also holds, the page is copied, all
layers and sequences of the step in one launch.  Each step uploads its own small
table, so steps in flight never see a later one's.  All calls of one cache
belong on one stream (or on streams that the caller orders).
"""
from __future__ import annotations

import heapq
import weakref
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..ops import paged
from ..ops.rotary import Rotary


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a step needs; nothing was changed."""


class PageTable:
    """Which pages each sequence holds, on the host."""

    def __init__(self, num_pages: int, page_size: int, max_len: Optional[int] = None):
        if num_pages < 1 or page_size < 1:
            raise ValueError("num_pages and page_size must be positive")
        if max_len is not None and max_len < 1:
            raise ValueError("max_len must be positive")
        self.num_pages = num_pages
        self.page_size = page_size
        self.max_len = max_len
        self._free = list(range(num_pages))  # a heap: the lowest free page first
        self._holders = [0] * num_pages
        self._pages: Dict[int, List[int]] = {}
        self._len: Dict[int, int] = {}
        self._next = 0

    def _known(self, seq: int) -> None:
        if seq not in self._pages:
            raise KeyError(f"no sequence {seq}")

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> List[int]:
        return list(self._pages)

    def length(self, seq: int) -> int:
        self._known(seq)
        return self._len[seq]

    def pages(self, seq: int) -> Tuple[int, ...]:
        self._known(seq)
        return tuple(self._pages[seq])

    def new(self) -> int:
        seq = self._next
        self._next += 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def _drop(self, page: int) -> None:
        self._holders[page] -= 1
        if self._holders[page] == 0:
            heapq.heappush(self._free, page)

    def free(self, seq: int) -> None:
        self._known(seq)
        for page in self._pages.pop(seq):
            self._drop(page)
        del self._len[seq]

    def fork(self, seq: int) -> int:
        """A new sequence that holds the same pages."""
        self._known(seq)
        new = self.new()
        # pages behind the length (reserved, not committed) are not shared
        keep = -(-self._len[seq] // self.page_size)
        self._pages[new] = self._pages[seq][:keep]
        self._len[new] = self._len[seq]
        for page in self._pages[new]:
            self._holders[page] += 1
        return new

    def truncate(self, seq: int, length: int) -> None:
        self._known(seq)
        if not 0 <= length <= self._len[seq]:
            raise ValueError(f"length {length} of a sequence of {self._len[seq]}")
        keep = -(-length // self.page_size)
        for page in self._pages[seq][keep:]:
            self._drop(page)
        del self._pages[seq][keep:]
        self._len[seq] = length

    def reserve(self, seqs: Sequence[int], counts: Sequence[int]) -> Tuple[List[int], List[int]]:
        """Room for ``counts[i]`` tokens behind each sequence, in pages that it alone
        holds.  Returns the copies (source pages, destination pages) that make the
        shared ones its own.  Raises, changing nothing, when it cannot."""
        if len(seqs) != len(counts):
            raise ValueError(f"{len(seqs)} sequences, {len(counts)} counts")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is twice in the step")
        need = 0
        private: Dict[int, int] = {}  # holders that would be left as pages are copied away
        plan = []
        for seq, n in zip(seqs, counts):
            self._known(seq)
            if n < 0:
                raise ValueError(f"{n} tokens")
            end = self._len[seq] + n
            if self.max_len is not None and end > self.max_len:
                raise ValueError(f"sequence {seq} would reach {end} tokens of {self.max_len}")
            have = len(self._pages[seq])
            first = self._len[seq] // self.page_size  # the page of the first new token
            copies = []
            if n > 0:
                for i in range(first, have):
                    page = self._pages[seq][i]
                    if private.get(page, self._holders[page]) > 1:
                        private[page] = private.get(page, self._holders[page]) - 1
                        copies.append(i)
            fresh = max(0, -(-end // self.page_size) - have) if n > 0 else 0
            need += fresh + len(copies)
            plan.append((seq, copies, fresh))
        if need > len(self._free):
            raise OutOfPages(f"{need} pages needed, {len(self._free)} free")
        src: List[int] = []
        dst: List[int] = []
        for seq, copies, fresh in plan:
            pages = self._pages[seq]
            for i in copies:
                page = heapq.heappop(self._free)
                self._holders[page] = 1
                # only tokens below the length are worth a copy
                if i * self.page_size < self._len[seq]:
                    src.append(pages[i])
                    dst.append(page)
                self._holders[pages[i]] -= 1  # others hold it still
                pages[i] = page
            for _ in range(fresh):
                page = heapq.heappop(self._free)
                self._holders[page] = 1
                pages.append(page)
        return src, dst

    def grow(self, seq: int, count: int) -> None:
        """Count ``count`` reserved tokens as held; pages behind them are given back."""
        self._known(seq)
        if count < 0 or -(-(self._len[seq] + count) // self.page_size) > len(self._pages[seq]):
            raise ValueError(f"{count} tokens are not reserved for sequence {seq}")
        self._len[seq] += count
        keep = -(-self._len[seq] // self.page_size)
        for page in self._pages[seq][keep:]:
            self._drop(page)
        del self._pages[seq][keep:]

    def compact(self) -> Tuple[List[int], List[int]]:
        """Moves that bring every held page below the number of pages in use."""
        used = self.num_pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.num_pages) if self._holders[p] > 0]
        to = dict(zip(high, holes))
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._holders[b], self._holders[a] = self._holders[a], 0
        self._free = list(range(used, self.num_pages))
        return high, holes


class CacheStep:
    """One call's worth of new tokens: page table, cached lengths and borders on the GPU."""

    def __init__(self, cache: "PagedKVCache", seqs: Sequence[int], counts: Sequence[int]):
        self.cache = cache
        self.seqs, self.counts = list(seqs), [int(n) for n in counts]
        table = cache.table
        if not self.seqs:
            raise ValueError("a step needs a sequence")
        cache._no_capture()
        for s in self.seqs:
            other = cache._open.get(s, lambda: None)()
            if other is not None and other._open:
                raise RuntimeError(f"sequence {s} has a step that is neither committed, accepted "
                                   "nor cancelled")
        src, dst = table.reserve(self.seqs, self.counts)
        if src:
            paged.copy_pages(cache.k, cache.v, src, dst)
        self.lengths = [table.length(s) for s in self.seqs]
        self.tokens = sum(self.counts)
        self.max_q = max(max(self.counts), 1)
        pages = [table.pages(s) for s in self.seqs]
        b, width = len(self.seqs), max(1, max(len(p) for p in pages))
        host = torch.zeros(b * (width + 2) + 1, dtype=torch.int32)
        grid = host[2 * b + 1:].view(b, width)
        for i, p in enumerate(pages):
            grid[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        host[:b] = torch.tensor(self.lengths, dtype=torch.int32)
        host[b + 1:2 * b + 1] = torch.tensor(self.counts, dtype=torch.int32).cumsum(0)
        dev = cache._upload(host)
        self.context_lens = dev[:b]
        self.cu_q = dev[b:2 * b + 1]
        self.block_table = dev[2 * b + 1:].view(b, width)
        self._open = True
        self._moves = cache._moves
        for s in self.seqs:
            cache._open[s] = weakref.ref(self)

    def _layer(self, layer: int) -> Tuple[torch.Tensor, torch.Tensor]:
        if not self._open:
            raise RuntimeError("the step is committed")
        if self._moves != self.cache._moves:
            raise RuntimeError("the cache was defragmented: the step's table is out of date")
        return self.cache.k[layer], self.cache.v[layer]

    def _rows(self, **tensors: Optional[torch.Tensor]) -> None:
        """Every token of the step has a row; rows behind them (a padded batch) are left."""
        for name, t in tensors.items():
            if t is not None and t.shape[0] < self.tokens:
                raise ValueError(f"{name} has {t.shape[0]} rows, the step {self.tokens} tokens")

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rotary: Optional[Rotary] = None,
               q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None):
        """Write the step's K (rotated) and V of one layer; returns q rotated, if given."""
        kp, vp = self._layer(layer)
        self._rows(k=k, v=v, q=q)
        if rotary is None:
            return paged.append_kv(k, v, kp, vp, self.block_table, self.context_lens, self.cu_q,
                                   positions=positions, q=q, status=status)
        return paged.append_kv(k, v, kp, vp, self.block_table, self.context_lens, self.cu_q,
                               positions=positions, inv_freq=rotary.inv_freq,
                               interleaved=rotary.interleaved, scale=rotary.scale, q=q,
                               status=status)

    def attend(self, layer: int, q: torch.Tensor, mask: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, return_lse: bool = False,
               out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
        """Attention of the step's tokens over the cache (see `ops.paged.tree_attention`)."""
        kp, vp = self._layer(layer)
        self._rows(q=q)
        return paged.tree_attention(q, kp, vp, self.block_table, self.context_lens, self.cu_q,
                                    max_q=self.max_q, mask=mask, scale=scale,
                                    return_lse=return_lse, out=out, status=status)

    def tree(self, parents: Sequence[Sequence[int]]) -> Tuple[torch.Tensor, torch.Tensor]:
        """Mask and depths of drafted trees, one parent list per sequence of the step."""
        if [len(p) for p in parents] != self.counts:
            raise ValueError("one parent per token of the step is needed")
        for p in parents:
            for i, up in enumerate(p):
                if not -1 <= up < i:
                    raise ValueError(f"parent {up} of token {i} is no token before it")
        flat = torch.tensor([x for p in parents for x in p], dtype=torch.int32)
        return paged.tree_mask(self.cache._upload(flat), self.cu_q, max_q=self.max_q)

    def positions(self, depth: torch.Tensor) -> torch.Tensor:
        """Rotary positions of tree tokens: cached length plus depth (int32)."""
        return torch.repeat_interleave(self.context_lens, self.cu_q[1:] - self.cu_q[:-1],
                                       output_size=self.tokens) + depth

    def _close(self, kept: Sequence[int]) -> None:
        for seq, n in zip(self.seqs, kept):
            self.cache.table.grow(seq, n)
        self._open = False

    def commit(self) -> None:
        """Every token of the step stays."""
        self._layer(0)
        self._close(self.counts)

    def cancel(self) -> None:
        """No token of the step stays."""
        if self._open:
            self._close([0] * len(self.seqs))

    def accept(self, paths: Sequence[Sequence[int]]) -> None:
        """The tokens on each sequence's path (increasing places within its tree; may
        be empty) stay, in every layer; the others are dropped."""
        self._layer(0)
        if len(paths) != len(self.seqs):
            raise ValueError(f"{len(paths)} paths for {len(self.seqs)} sequences")
        for p, n in zip(paths, self.counts):
            if any(not 0 <= x < n for x in p) or any(b <= a for a, b in zip(p, list(p)[1:])):
                raise ValueError(f"path {list(p)} is not increasing within {n} tokens")
        width = max(len(p) for p in paths)
        if any(list(p) != list(range(len(p))) for p in paths):
            host = torch.zeros(len(paths), width + 1, dtype=torch.int32)
            for i, p in enumerate(paths):
                host[i, 0] = len(p)
                host[i, 1:1 + len(p)] = torch.tensor(list(p), dtype=torch.int32)
            dev = self.cache._upload(host)
            lens = dev[:, 0].contiguous()
            paged.compact_path(self.cache.k, self.cache.v, self.block_table, self.context_lens,
                               dev[:, 1:], lens)
        self._close([len(p) for p in paths])


class PagedKVCache:
    """Pools of K and V pages of every layer and the sequences that live in them.

    ``k`` and ``v`` are ``[layers, num_pages, heads_kv, page_size, head_dim]``.
    ``max_len`` bounds a sequence's tokens.
    """

    def __init__(self, layers: int, num_pages: int, heads_kv: int, head_dim: int,
                 page_size: int = 64, max_len: Optional[int] = None,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError("dtype must be bfloat16, float16 or float32")
        if layers < 1 or heads_kv < 1:
            raise ValueError("layers and heads_kv must be positive")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64, 128 or 256")
        self.table = PageTable(num_pages, page_size, max_len)
        shape = (layers, num_pages, heads_kv, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.device = self.k.device
        self._open: Dict[int, "weakref.ref[CacheStep]"] = {}  # each sequence's last step
        self._moves = 0

    def _no_capture(self) -> None:
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("tables, trees and paths are uploaded once: make the step, its tree "
                               "and its acceptance outside a capture")

    def _upload(self, host: torch.Tensor) -> torch.Tensor:
        """A small tensor of the host on the cache's device, without waiting for either."""
        if self.device.type == "cuda":
            self._no_capture()
            host = host.pin_memory()
        return host.to(self.device, non_blocking=True)

    def new_sequence(self) -> int:
        return self.table.new()

    def fork(self, seq: int) -> int:
        return self.table.fork(seq)

    def _idle(self, seq: int) -> None:
        step = self._open.get(seq, lambda: None)()
        if step is not None and step._open:
            raise RuntimeError(f"sequence {seq} has an open step: commit, accept or cancel it first")

    def free(self, seq: int) -> None:
        self._idle(seq)
        self.table.free(seq)
        self._open.pop(seq, None)

    def truncate(self, seq: int, length: int) -> None:
        """Drop the tokens of a sequence behind ``length``."""
        self._idle(seq)
        self.table.truncate(seq, length)

    def length(self, seq: int) -> int:
        return self.table.length(seq)

    def step(self, seqs: Sequence[int], counts: Sequence[int]) -> CacheStep:
        """Reserve room for ``counts[i]`` new tokens of each sequence."""
        return CacheStep(self, seqs, counts)

    def defragment(self) -> int:
        """Move the pages in use to the front of the pool; returns how many there are.
        No step may be open."""
        for seq in self.table.sequences():
            self._idle(seq)
        self._moves += 1
        src, dst = self.table.compact()
        if src:
            paged.copy_pages(self.k, self.v, src, dst)
        return self.table.num_pages - self.table.free_pages
