"""Plan of a decode batch kept alive across steps.

The reference rebuilds everything in every decode step: radix tree, tile plan, the per-bucket
tables and their host-to-device copies (``prefix_attn/async_tree.py:23-30``, cached once per
forward pass at ``plugin/vllm/attention/backends/prefix_attn.py:318-340`` and left stale by
``advance_step`` at ``:430-438``).  Between two steps of a running batch almost nothing changes:
every request is one token longer and now and then one page longer.  ``DecodePlanner.step`` first
tries to grow the previous step's tree and device work list in place (``PrefixTreeCPP.advance``:
item lengths and appended page ids are patched and the list is copied into the same device buffer)
and only falls back to a rebuild when the batch really changed.  Either way it returns a
``PrefixTreeCPP`` for ``prefix_attn_with_kvcache(q, k_cache, v_cache, tree, scale, out)``.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from ._prefix_attn import PrefixTreeCPP
from .beam import PagePool, beam_select
from .cache_ops import copy_pages


class DecodePlanner:
    def __init__(self, block_size: int, HRatio: int, kvHead: int, device: Union[torch.device, str],
                 MNWs: Optional[List[List[int]]] = None, semantics: str = "cpp", kv_cache_dtype: str = "auto"):
        self.block_size, self.hratio, self.kv_heads = int(block_size), int(HRatio), int(kvHead)
        self.device = torch.device(device)
        self.mnws, self.semantics = MNWs, semantics
        self.kv_cache_dtype = kv_cache_dtype    # "int4": plans for prefix_attn_with_int4_kvcache
        self.tree: Optional[PrefixTreeCPP] = None
        self.rebuilds = 0           # steps that built tree and work list from scratch
        self.advances = 0           # steps that grew them in place

    def step(self, seq_lens, block_table: torch.Tensor) -> PrefixTreeCPP:
        """``seq_lens``: list of ints or CPU int32 tensor; ``block_table``: padded CPU int32 tensor
        ``[num_seqs, max_blocks]`` (the arguments of ``build_radix_tree``).  Call it on the stream
        the attention runs on: an in-place update is copied to the device on the current stream."""
        if self.tree is not None and self.tree.advance(seq_lens, block_table):
            self.advances += 1
            return self.tree
        tree = PrefixTreeCPP(self.block_size, self.semantics)
        tree.build_radix_tree(seq_lens, block_table)
        tree.pack_schedule(self.mnws, self.hratio, self.kv_heads)
        tree.kernel_info.to_gpu(self.device, self.kv_cache_dtype)
        self.tree = tree
        self.rebuilds += 1
        return tree


class BeamPlanner(DecodePlanner):
    """A ``DecodePlanner`` for beam search: it also keeps the beams' pages.

    ``pool`` counts the pages of ``caches``, the paged caches of all layers (16-bit K and V tensors, or
    4-bit ones with ``kv_cache_dtype="int4"``).  Per step::

        slots = planner.extend()                    # where the new token of every beam goes
        tree = planner.plan()                       # plan of the attention that includes it
        ... append to slots, attend with tree, run the model ...
        scores, parents, tokens = planner.select(logits, scores)

    ``select`` keeps as many candidates as there are beams, forks the block tables and copies the
    part-filled pages in every cache.  Reading the parents waits for the selection."""

    def __init__(self, pool: PagePool, caches: Sequence[torch.Tensor], HRatio: int, kvHead: int,
                 device: Union[torch.device, str], kv_cache_dtype: str = "auto"):
        super().__init__(pool.page_size, HRatio, kvHead, device, kv_cache_dtype=kv_cache_dtype)
        self.pool, self.caches = pool, list(caches)
        self.tables: List[List[int]] = []
        self.lens: List[int] = []

    def begin(self, tables: Sequence[Sequence[int]], lens: Sequence[int]) -> None:
        """The beams of all batch entries, entry after entry; their pages were taken from the pool."""
        self.tables, self.lens = [list(t) for t in tables], [int(n) for n in lens]
        self.tree = None

    def extend(self) -> torch.Tensor:
        """Slots (int64, on the host) of the next token of every beam, whose lengths then include it."""
        need = sum(n % self.pool.page_size == 0 for n in self.lens)
        if need > self.pool.num_free:
            raise RuntimeError(f"the cache is full: {need} pages asked for, {self.pool.num_free} free")
        slots = [self.pool.extend(t, n) for t, n in zip(self.tables, self.lens)]
        self.lens = [n + 1 for n in self.lens]
        return torch.tensor(slots, dtype=torch.int64)

    def plan(self) -> PrefixTreeCPP:
        table = torch.zeros(len(self.tables), max((len(t) for t in self.tables), default=0), dtype=torch.int32)
        for i, t in enumerate(self.tables):
            table[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        return self.step(self.lens, table)

    def select(self, logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None,
               pad_token: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``logits [batch, beams, vocab]`` of the beams given to ``begin``; see ``beam_select``."""
        batch, beams = scores.shape
        if batch * beams != len(self.tables):
            raise RuntimeError("scores must be [batch, beams] of the beams in the tables")
        out = beam_select(logits, scores, beams, finished, pad_token)
        rows = (out[1].cpu().to(torch.int64) + torch.arange(batch)[:, None] * beams).flatten().tolist()
        self.tables, self.lens, pairs = self.pool.fork(self.tables, self.lens, rows)
        copy_pages(self.caches, pairs)
        return out
