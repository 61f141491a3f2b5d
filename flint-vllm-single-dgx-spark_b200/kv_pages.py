"""The pages of the KV cache as a pool that streams share: reserve, fork, free, compact.

The cache of all layers is one bf16 tensor ``kv`` [layers, blocks, kv_heads, 16, 256]; the pool's state is int32 tensors on
the device: ``ref`` [blocks] (how many streams hold a page, 0: free), ``block_tables`` [streams, max_blocks] (-1 behind a
stream's pages), ``seq_lens`` and ``num_pages`` [streams].  Every call runs on the current stream without reading anything
back; pages come from the lowest free ids in the order of the call's streams, so equal states give equal results.  A
request that does not fit is left out whole and recorded in the device status (``_lib.check_device_status``); behind the
first that finds too few free pages, every later one of the call that needs a page is refused too.

* ``flint_kv_reserve(ref, block_tables, seq_lens, num_pages, streams, lens)`` -- room for lens[i] tokens in streams[i]
  (seq_lens is there so that the pool's state can be passed as one; it is neither read nor written)
* ``flint_kv_fork(kv, ref, block_tables, seq_lens, num_pages, src, dst)`` -- the empty stream dst[i] becomes a copy of
  src[i]: whole pages shared, the last page copied in every layer if it is not full
* ``flint_kv_free(ref, block_tables, seq_lens, num_pages, streams)`` -- a stream named twice is freed once
* ``flint_kv_compact(kv, ref, block_tables, num_pages, remap, live)`` -- used pages to the ids 0 .. live - 1;
  remap int32 [blocks] tells where a used page went (-1: free), live int32 [1] their number (num_pages is not read)

``PagePool`` keeps the tensors of one cache together.
"""
from __future__ import annotations

import torch

from . import _lib
from . import ops as _ops


def flint_kv_reserve(ref, block_tables, seq_lens, num_pages, streams, lens):
    _ops.run("kv_reserve", ref, block_tables, num_pages, streams, lens)


def flint_kv_fork(kv, ref, block_tables, seq_lens, num_pages, src, dst):
    _ops.run("kv_fork", kv, ref, block_tables, seq_lens, num_pages, src, dst)


def flint_kv_free(ref, block_tables, seq_lens, num_pages, streams):
    _ops.run("kv_free", ref, block_tables, seq_lens, num_pages, streams)


def flint_kv_compact(kv, ref, block_tables, num_pages, remap, live):
    _ops.run("kv_compact", kv, ref, block_tables, num_pages, remap, live)


class PagePool:
    """An empty pool over the cache ``kv`` for ``streams`` streams of up to ``max_blocks`` pages each."""

    def __init__(self, kv: torch.Tensor, streams: int, max_blocks: int):
        _lib.require_cuda(kv, "PagePool")
        if streams < 1 or max_blocks < 1:
            raise ValueError("PagePool needs at least one stream and one page per stream")
        self.kv = kv
        new = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=kv.device)
        self.ref, self.seq_lens, self.num_pages = new(kv.shape[1]), new(streams), new(streams)
        self.block_tables = new(streams, max_blocks).fill_(-1)
        self.remap, self.live = new(kv.shape[1]), new(1)

    def _ids(self, ids) -> torch.Tensor:
        if isinstance(ids, torch.Tensor):
            return ids
        return torch.tensor(ids, dtype=torch.int32, device=self.kv.device)

    @property
    def state(self):
        return self.ref, self.block_tables, self.seq_lens, self.num_pages

    def reserve(self, streams, lens) -> None:
        flint_kv_reserve(*self.state, self._ids(streams), self._ids(lens))

    def fork(self, src, dst) -> None:
        flint_kv_fork(self.kv, *self.state, self._ids(src), self._ids(dst))

    def free(self, streams) -> None:
        flint_kv_free(*self.state, self._ids(streams))

    def compact(self) -> torch.Tensor:
        """-> remap (this pool's buffer, rewritten by the next call)."""
        flint_kv_compact(self.kv, self.ref, self.block_tables, self.num_pages, self.remap, self.live)
        return self.remap
