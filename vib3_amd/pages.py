"""The pages of a paged cache, forked and compacted in all layers at once (host side, torch for memory).

``fork_pages`` lets sequences go on from another's tokens: they share its full pages and get a copy of the last one.
``PageCompaction`` moves the pages in use to the front of the pools and rewrites the block table, which frees whatever no sequence
refers to any more. Both take the layers' caches, all GqaCache or MlaCache of one device with the same number and size of pages and
one block table. The C ABI and what each of them does are in include/vib3_hip.h. Every call runs on the current torch stream of the
tensors' device; there is no CPU branch.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _lib
from .gqa import GqaCache
from .mla import _INT, MlaCache, _dims, _flat, _launch

Cache = Union[GqaCache, MlaCache]


def _pools(caches: Sequence[Cache]):
    """The caches' pools as an array for the C ABI, the number and size of their pages, their device and an owner of it."""
    pools, kind = [], None
    for c in caches:
        if isinstance(c, GqaCache):
            tensors, kv_heads, size = (c.keys, c.values), c.kv_heads, c.keys.element_size()
            pages, page_size, _, dim = c.keys.shape
            page, token, head, _ = c.keys.stride()
            # tokens with all of their heads in one run of bytes, or a run of tokens for each head
            run = (0, token * size, 1, kv_heads * dim * size) if kv_heads == 1 or head == dim else \
                (head * size, token * size, kv_heads, dim * size)
        elif isinstance(c, MlaCache):
            tensors, size = (c.pool,), c.pool.element_size()
            pages, page_size, width = c.pool.shape
            page, token, _ = c.pool.stride()
            run = (0, token * size, 1, width * size)
        else:
            raise TypeError(f"caches must be GqaCache or MlaCache objects, not {type(c).__name__}")
        if kind is None:
            kind = (pages, page_size, c.index)
        elif kind != (pages, page_size, c.index):
            raise ValueError(f"caches of (pages, page size, device) {kind} and {(pages, page_size, c.index)} in one call")
        pools += [_lib.PagePoolDesc(t.data_ptr(), page * size, *run) for t in tensors]
    if kind is None:
        raise ValueError("no caches")
    return (_lib.PagePoolDesc * len(pools))(*pools), kind


def fork_pages(caches: Sequence[Cache], block_table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, children: torch.Tensor,
               new_pages: torch.Tensor) -> None:
    """Let sequence children[i] go on from the first lens[parents[i]] tokens of sequence parents[i] (vib3_launch_fork_pages).

    Row children[i] of block_table (int32 [num_seqs, max_pages]) becomes the parent's full pages, then new_pages[i], then -1; the
    tokens of the parent's last page, if that is not full, are copied to new_pages[i] in every cache. parents, children and
    new_pages are int32 [count]; lens (int32 [num_seqs]) is read only."""
    pools, (pages, page_size, index) = _pools(caches)
    seqs, width = _dims(block_table, "block_table", (_INT,), 2)
    count = _dims(parents, "parents", (_INT,), 1)[0]
    a = _lib.ForkPagesDesc(pools, len(pools), pages, page_size, _flat(block_table, "block_table", _INT, (seqs, width), index), seqs, width,
                           _flat(lens, "lens", _INT, (seqs,), index), count,
                           *(_flat(t, n, _INT, (count,), index) for t, n in ((parents, "parents"), (children, "children"),
                                                                             (new_pages, "new_pages"))))
    _launch("vib3_launch_fork_pages", a, index)


class PageCompaction:
    """Moves the pages in use to the front of the caches' pools: owns the workspace. Launches that may overlap (other streams,
    captured graphs) need a PageCompaction each."""

    def __init__(self, caches: Sequence[Cache]):
        self.caches = list(caches)
        self._pools, (self.num_pages, self.page_size, self.index) = _pools(self.caches)
        n = _lib.load().vib3_compact_pages_workspace_bytes(_lib.CompactPagesDesc(num_pages=self.num_pages))
        if n == 0:
            raise ValueError(f"PageCompaction: unsupported number of pages {self.num_pages}")
        device = torch.device("cuda", self.index)
        self.workspace = torch.empty(n + 256, dtype=torch.uint8, device=device)
        self.live = torch.zeros(1, dtype=_INT, device=device)
        self._space = ((self.workspace.data_ptr() + 255) // 256 * 256, n)

    def launch(self, block_table: torch.Tensor, lens: torch.Tensor, out_table: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Compact the pages of the sequences' first lens[s] tokens (int32 [num_seqs]; block_table int32 [num_seqs, max_pages])
        and write the table with the new numbers to out_table (default: in place), -1 in entries that no token uses. Pages
        that only such entries named are free from then on. Returns self.live (int32 [1], on the device): the number of
        pages in use; pages from there on are free (vib3_launch_compact_pages)."""
        seqs, width = _dims(block_table, "block_table", (_INT,), 2)
        at = _flat(block_table, "block_table", _INT, (seqs, width), self.index)
        to = at if out_table is None else _flat(out_table, "out_table", _INT, (seqs, width), self.index)
        a = _lib.CompactPagesDesc(self._pools, len(self._pools), self.num_pages, self.page_size, at, seqs, width,
                                  _flat(lens, "lens", _INT, (seqs,), self.index), to, self.live.data_ptr(), *self._space)
        _launch("vib3_launch_compact_pages", a, self.index)
        return self.live
