"""Moving whole KV blocks between a host-side cache and the device cache (block swap for
preemption / offload).  Same call surface and no-op rules as ``copy_kv_blocks`` in tt-xla's
``integrations/vllm_plugin/vllm_tt/model_runner.py:5433-5474``: caches are dicts
``layer name -> tensor`` or ``layer name -> (k_cache, v_cache)`` with blocks on dim 0 (an
8-bit layer: all of its kv_cache, scales and key bounds too), and block ``src_block_ids[i]``
of every source tensor lands in block ``dst_block_ids[i]`` of the matching destination
tensor.  Pure block copies: torch's gather / scatter on dim 0 plus one transfer per tensor;
nothing is computed.

``copy_cache_blocks`` copies blocks inside the device caches of all layers, one call of
``tt::copy_cache_blocks_``; ``CachePages`` is the host's account of a cache's blocks: which
sequence holds which, which of them are shared, and the copies that forks, writes and
compaction want.
"""

from __future__ import annotations

import heapq
from typing import Dict, Hashable, Iterable, List, Literal, Sequence, Tuple, Union

import torch

from . import media_ops  # noqa: F401  (registers the operator)

Cache = Union[torch.Tensor, Sequence[torch.Tensor]]


def _device_of(value: Cache) -> torch.device:
    return value[0].device if isinstance(value, (list, tuple)) else value.device


def _move(src: torch.Tensor, dst: torch.Tensor, src_idx: torch.Tensor, dst_idx: torch.Tensor) -> None:
    if src.dtype == dst.dtype and src.dtype.itemsize == 1:  # (torch gathers and scatters bytes everywhere, 8-bit floats not on the host)
        src, dst = src.view(torch.uint8), dst.view(torch.uint8)
    picked = src.index_select(0, src_idx)
    dst.index_copy_(0, dst_idx, picked.to(dst.device, non_blocking=False))


def copy_kv_blocks(
    src_kv_caches: Dict[str, Cache],
    dst_kv_caches: Dict[str, Cache],
    src_block_ids: List[int],
    dst_block_ids: List[int],
    direction: Literal["h2d", "d2h"],
) -> None:
    if (
        not src_kv_caches
        or not dst_kv_caches
        or not src_block_ids
        or not dst_block_ids
        or len(src_block_ids) != len(dst_block_ids)
    ):
        return
    if direction not in ("h2d", "d2h"):
        raise ValueError(f"direction must be 'h2d' or 'd2h', got {direction!r}")
    src_device = _device_of(next(iter(src_kv_caches.values())))
    dst_device = _device_of(next(iter(dst_kv_caches.values())))
    src_idx = torch.tensor(src_block_ids, dtype=torch.int64, device=src_device)
    dst_idx = torch.tensor(dst_block_ids, dtype=torch.int64, device=dst_device)
    for name, src in src_kv_caches.items():
        dst = dst_kv_caches[name]
        if isinstance(src, (list, tuple)):
            if len(src) != len(dst):
                raise ValueError(f"layer {name!r} has {len(src)} tensors on one side and {len(dst)} on the other")
            for s, d in zip(src, dst):
                _move(s, d, src_idx, dst_idx)
        else:
            _move(src, dst, src_idx, dst_idx)


def copy_cache_blocks(kv_caches: Dict[str, Cache], pairs: Sequence[Tuple[int, int]]) -> None:
    """Copies block ``source`` to block ``target`` in every tensor of every layer, as if the pairs (source, target) went one after the
    other.  Tensors that several layers share (one layer's cache written by another's) are copied once."""
    if not pairs or not kv_caches:
        return
    tensors: Dict[int, torch.Tensor] = {}
    for value in kv_caches.values():
        for t in value if isinstance(value, (list, tuple)) else (value,):
            if t.numel():
                tensors[t.data_ptr()] = t
    if not tensors:
        return
    some = list(tensors.values())
    nb = min(t.shape[0] for t in some)
    for pair in pairs:
        if not all(0 <= b < nb for b in pair):
            raise ValueError(f"block pair {tuple(pair)} is outside a cache of {nb} blocks")
    ids = torch.tensor(list(pairs), dtype=torch.int32).t().contiguous().to(some[0].device)
    torch.ops.tt.copy_cache_blocks_(some, ids[0], ids[1])


class CachePages:
    """Who holds which blocks ("pages") of a paged cache.

    Sequences grow page by page, may share pages (``fork``) and give them back (``free``, ``truncate``).  A page that is about to be written
    while others hold it, too, is replaced by a copy; the calls that lead to writes answer with the pairs (source, target) to copy first
    (``copy_cache_blocks``).  Host bookkeeping alone: nothing here touches a device.

    reserved  pages that are nobody's: the first ones (block 0 is the null block of :class:`~tt_xla_amd.metadata.PagedMetadataBuilder`).
    """

    def __init__(self, num_blocks: int, block_size: int, reserved: int = 1):
        if num_blocks <= 0 or block_size <= 0 or not 0 <= reserved <= num_blocks:
            raise ValueError(f"{num_blocks} blocks of {block_size} with {reserved} reserved")
        self.num_blocks, self.block_size, self.reserved = num_blocks, block_size, reserved
        self._free = list(range(reserved, num_blocks))  # a heap: the lowest is taken next
        self._holders = [0] * num_blocks
        self._pages: Dict[Hashable, List[int]] = {}
        self._length: Dict[Hashable, int] = {}

    # ---- questions ----
    def length(self, sequence: Hashable) -> int:
        return self._length[sequence]

    def pages(self, sequence: Hashable) -> List[int]:
        return list(self._pages[sequence])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def table(self, sequences: Iterable[Hashable], width: int, fill: int = 0) -> torch.Tensor:
        """[sequences, width] int32 page table."""
        rows = [self._pages[s] for s in sequences]
        out = torch.full((len(rows), width), fill, dtype=torch.int32)
        for i, pages in enumerate(rows):
            if len(pages) > width:
                raise ValueError(f"a sequence of {len(pages)} pages does not fit a table of {width} columns")
            out[i, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
        return out

    # ---- changes ----
    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise RuntimeError(f"{n} pages wanted, {len(self._free)} free")
        pages = [heapq.heappop(self._free) for _ in range(n)]
        for p in pages:
            self._holders[p] = 1
        return pages

    def _release(self, pages: Iterable[int]) -> None:
        for p in pages:
            self._holders[p] -= 1
            if self._holders[p] == 0:
                heapq.heappush(self._free, p)

    def _own(self, sequence: Hashable, first: int, end: int, grow_to: int) -> List[Tuple[int, int]]:
        """Makes pages of positions [first, end) the sequence's own and appends pages up to ``grow_to``; all or nothing."""
        pages, bs = self._pages[sequence], self.block_size
        shared = [i for i in range(first // bs, min(-(-end // bs), len(pages))) if self._holders[pages[i]] > 1] if end > first else []
        fresh = self._take(len(shared) + max(0, -(-grow_to // bs) - len(pages)))
        pairs = []
        for i in shared:
            new = fresh.pop(0)
            pairs.append((pages[i], new))
            self._release([pages[i]])
            pages[i] = new
        pages.extend(fresh)
        return pairs

    def add(self, sequence: Hashable, tokens: int) -> None:
        """A new sequence with room for ``tokens`` tokens."""
        if sequence in self._pages:
            raise ValueError(f"sequence {sequence!r} is there already")
        if tokens < 0:
            raise ValueError("a sequence has no fewer than zero tokens")
        pages = self._take(-(-tokens // self.block_size))
        self._pages[sequence], self._length[sequence] = pages, tokens

    def extend(self, sequence: Hashable, tokens: int) -> List[Tuple[int, int]]:
        """``tokens`` more, about to be written behind the last one; the pairs to copy before."""
        if tokens < 0:
            raise ValueError("a sequence is extended by no fewer than zero tokens")
        n = self._length[sequence]
        pairs = self._own(sequence, n, n + tokens, n + tokens)
        self._length[sequence] = n + tokens
        return pairs

    def fork(self, sequence: Hashable, child: Hashable) -> None:
        """A second sequence of the same tokens, on the same pages."""
        if child in self._pages:
            raise ValueError(f"sequence {child!r} is there already")
        self._pages[child], self._length[child] = list(self._pages[sequence]), self._length[sequence]
        for p in self._pages[child]:
            self._holders[p] += 1

    def own(self, sequence: Hashable, first: int = 0) -> List[Tuple[int, int]]:
        """The pages from position ``first`` on, about to be written (``tt::keep_cache_tokens_``); the pairs to copy before."""
        if first < 0:
            raise ValueError("positions start at zero")
        return self._own(sequence, first, self._length[sequence], 0)

    def truncate(self, sequence: Hashable, tokens: int) -> None:
        """The first ``tokens`` tokens stay; pages behind them go back."""
        if not 0 <= tokens <= self._length[sequence]:
            raise ValueError(f"sequence {sequence!r} has {self._length[sequence]} tokens, not {tokens}")
        keep = -(-tokens // self.block_size)
        self._release(self._pages[sequence][keep:])
        del self._pages[sequence][keep:]
        self._length[sequence] = tokens

    def free(self, sequence: Hashable) -> None:
        self._release(self._pages.pop(sequence))
        del self._length[sequence]

    def compact(self) -> List[Tuple[int, int]]:
        """Moves the pages in use to the lowest ids, so that all behind them are free; the pairs to copy, in order."""
        used = [p for p in range(self.reserved, self.num_blocks) if self._holders[p]]
        end = self.reserved + len(used)
        holes = [p for p in range(self.reserved, end) if not self._holders[p]]
        moved = dict(zip([p for p in used if p >= end], holes))
        for old, new in moved.items():
            self._holders[new], self._holders[old] = self._holders[old], 0
        for pages in self._pages.values():
            pages[:] = [moved.get(p, p) for p in pages]
        self._free = list(range(end, self.num_blocks))
        return list(moved.items())
