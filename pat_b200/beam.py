"""Beam (tree) search over a paged cache: choosing the next beams, and the pages they hold.

The reference leaves both to its serving engine; its deep-tree workloads are the batches such a
search produces.  ``beam_select`` is this library's kernel on PyTorch's current stream; ``PagePool`` is
host bookkeeping like the radix tree, since the plan of a step is made on the host from its block tables.
"""
from __future__ import annotations

import struct
from operator import index as index_of
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native as N
from ._launch import Signatures, launch, strides_of, struct_tail

_LOGIT_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num_out: int, finished: Optional[torch.Tensor] = None,
                pad_token: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``num_out`` best continuations of every batch entry, over its beams and the vocabulary.

    ``logits [batch, beams, vocab]`` (fp32, bf16 or fp16; any batch and beam strides, the last dimension
    contiguous), ``scores [batch, beams]`` fp32: the beams' log-probabilities so far.  The value of
    token ``v`` after beam ``k`` is ``scores[b, k] + log_softmax(logits[b, k])[v]``.  ``finished
    [batch, beams]`` (bool): such a beam has one candidate, ``pad_token`` with its score unchanged.

    Returns ``(scores fp32, parents int32, tokens int32)``, each ``[batch, num_out]``: larger values
    first, ties to the lower beam, then the lower token.  A beam whose score is not finite (the beams
    beyond the first of a search that starts), or whose logits hold a NaN or +inf or nothing but -inf, takes no
    part; where an entry has fewer finite values than ``num_out``, -inf entries follow, lowest beam and
    token first.  ``num_out`` <= 128, ``beams`` <= 512, ``vocab`` <= 2^24."""
    num_out, pad_token = index_of(num_out), index_of(pad_token)
    sig = (logits.dtype, logits.shape, logits.stride(), logits.get_device(), scores.dtype, scores.shape, scores.stride(),
           scores.get_device(), num_out, pad_token)
    if finished is not None:
        sig += (finished.dtype, finished.shape, finished.stride(), finished.get_device())
    known = _beam_calls.get(sig)
    if known is None:
        known = _beam_calls.remember(sig, _check_beam(logits, scores, num_out, finished, pad_token))
    tail, index, batch, num_out, need, dense_scores, dense_finished = known
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return beam_select(logits, scores, num_out, finished, pad_token)
    dev = logits.device
    out_scores = torch.empty(batch, num_out, dtype=torch.float32, device=dev)
    out_parents = torch.empty(batch, num_out, dtype=torch.int32, device=dev)
    out_tokens = torch.empty(batch, num_out, dtype=torch.int32, device=dev)
    if batch == 0:
        return out_scores, out_parents, out_tokens
    if not dense_scores:
        scores = scores.contiguous()
    if not dense_finished:
        finished = finished.contiguous()
    # Scratch: calls on one stream run one after the other and share it; a captured call gets its own, which belongs to
    # the graph, since graphs captured on one stream may be replayed on several.
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    else:
        key = (index, torch._C._cuda_getCurrentRawStream(index))
        ws = _beam_scratch.get(key)
        if ws is None or ws.numel() < need:
            ws = _beam_scratch[key] = torch.empty(need, dtype=torch.uint8, device=dev)
    rc = launch(N.load().pat_b200_beam_select,
                _BEAM_POINTERS.pack(logits.data_ptr(), scores.data_ptr(), finished.data_ptr() if finished is not None else 0,
                                    out_scores.data_ptr(), out_parents.data_ptr(), out_tokens.data_ptr(), ws.data_ptr()) + tail, index)
    if rc != 0:
        raise RuntimeError(f"beam_select failed: {N.strerror(rc)} ({rc})")
    return out_scores, out_parents, out_tokens


_BEAM_POINTERS = struct.Struct("7P")
_beam_calls = Signatures()
_beam_scratch = {}         # (device, stream) -> workspace


def _check_beam(logits, scores, num_out, finished, pad_token):
    for name, t in (("logits", logits), ("scores", scores), ("finished", finished)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if t.device != logits.device:
            raise RuntimeError(f"{name} must be on the device of logits")
    if logits.dtype not in _LOGIT_DTYPES:
        raise RuntimeError("logits must be fp32, bf16 or fp16")
    if logits.dim() != 3:
        raise RuntimeError("logits must be [batch, beams, vocab]")
    batch, beams, vocab = logits.shape
    if scores.dtype != torch.float32 or tuple(scores.shape) != (batch, beams):
        raise RuntimeError("scores must be float32 [batch, beams]")
    if finished is not None and (finished.dtype not in (torch.bool, torch.uint8) or tuple(finished.shape) != (batch, beams)):
        raise RuntimeError("finished must be bool [batch, beams]")
    if beams < 1 or vocab < 1:
        raise RuntimeError("logits must hold at least one beam and one token")
    if not 1 <= int(num_out) <= beams * vocab:
        raise RuntimeError("num_out must be between 1 and beams * vocab")
    if not 0 <= int(pad_token) < vocab:
        raise RuntimeError("pad_token must be a token of the vocabulary")
    if vocab > 1 and logits.stride(2) != 1:
        raise RuntimeError("logits must have a contiguous last dimension")
    need = N.load().pat_b200_beam_workspace_bytes(max(batch, 1), beams, vocab, int(num_out))
    if need == 0:
        raise RuntimeError("beam_select supports num_out <= 128, beams <= 512 and vocab <= 2^24")
    dense_scores = beams == 1 or scores.stride(1) == 1
    dense_finished = finished is None or beams == 1 or finished.stride(1) == 1
    a = N.BeamArgs()
    a.logits_batch_stride, a.logits_beam_stride = strides_of(logits)[:2]
    a.scores_batch_stride = strides_of(scores)[0] if dense_scores else beams
    a.finished_batch_stride = 0 if finished is None else strides_of(finished)[0] if dense_finished else beams
    a.batch, a.beams, a.vocab, a.num_out = batch, beams, vocab, int(num_out)
    a.dtype, a.pad_token = _LOGIT_DTYPES[logits.dtype], int(pad_token)
    a.workspace_bytes = need
    return struct_tail(a, _BEAM_POINTERS.size), logits.get_device(), batch, int(num_out), need, dense_scores, dense_finished


class PagePool:
    """Which pages of a paged cache are in use, and by how many requests.

    Block tables are lists of page ids, one per request; a request of ``length`` tokens holds
    ``ceil(length / page_size)`` pages.  Full pages may belong to several requests; the part-filled last
    page, which the next token is written into, belongs to one.  Plans that move pages come back as
    ``(from, to)`` pairs for ``cache_ops.copy_pages``; run them before the next token is appended."""

    def __init__(self, num_pages: int, page_size: int):
        if num_pages < 0 or page_size < 1:
            raise ValueError("num_pages and page_size must be positive")
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.uses = np.zeros(self.num_pages, dtype=np.int64)

    @property
    def num_free(self) -> int:
        return int((self.uses == 0).sum())

    def alloc(self, count: int) -> List[int]:
        """``count`` free pages, lowest ids first."""
        if count < 0:
            raise ValueError("count must not be negative")
        free = np.flatnonzero(self.uses == 0)[:count]
        if len(free) < count:
            raise RuntimeError(f"the cache is full: {count} pages asked for, {len(free)} free")
        self.uses[free] += 1
        return free.tolist()

    def share(self, pages: Sequence[int]) -> None:
        """One more request holds these (full) pages."""
        rows = self._in_use(pages)
        np.add.at(self.uses, rows, 1)

    def free(self, pages: Sequence[int]) -> None:
        """A request gives its pages back; a page is free once nobody holds it."""
        rows = self._in_use(pages)
        less = np.bincount(rows, minlength=self.num_pages)
        if (less > self.uses).any():
            raise RuntimeError("a page is freed more often than it is held")
        self.uses -= less

    def _in_use(self, pages) -> np.ndarray:
        rows = np.asarray(list(pages), dtype=np.int64)
        if rows.size and (rows.min() < 0 or rows.max() >= self.num_pages):
            raise RuntimeError("page outside the cache")
        if rows.size and (self.uses[rows] == 0).any():
            raise RuntimeError("page is not in use")
        return rows

    def extend(self, table: List[int], length: int) -> int:
        """Room for one more token behind ``length`` tokens: appends a page to ``table`` where the last one
        is full, and returns the token's slot."""
        if length % self.page_size == 0:
            table.extend(self.alloc(1))
        return table[length // self.page_size] * self.page_size + length % self.page_size

    def fork(self, tables: Sequence[Sequence[int]], lens: Sequence[int], parents: Sequence[int]
             ) -> Tuple[List[List[int]], List[int], List[Tuple[int, int]]]:
        """The requests that follow: number ``i`` continues ``parents[i]``.  Full pages are shared; of a
        part-filled last page the first child takes the original and every other one a copy.  Requests
        nobody continues give their pages back.  Returns ``(tables, lens, pairs)``; a copy's target was free
        before the call, so targets are never sources.  Raises, with nothing changed, when there are too
        few free pages."""
        tables = [list(t) for t in tables]
        parents = [int(p) for p in parents]
        if len(lens) != len(tables) or any(n < 0 or len(t) * self.page_size < n for t, n in zip(tables, lens)):
            raise RuntimeError("lens must give every table a length that its pages hold")
        for t in tables:
            self._in_use(t)
        for p in parents:
            if not 0 <= p < len(tables):
                raise RuntimeError("parent outside the batch")
        seen, split = set(), []
        for p in parents:
            split.append(lens[p] % self.page_size != 0 and p in seen)
            seen.add(p)
        fresh = iter(self.alloc(sum(split)))
        out, pairs = [], []
        for p, needs_copy in zip(parents, split):
            row = tables[p][:-(-lens[p] // self.page_size)]
            if needs_copy:
                page = next(fresh)
                pairs.append((row[-1], page))
                self.share(row[:-1])
                row = row[:-1] + [page]
            else:
                self.share(row)
            out.append(row)
        for t in tables:
            self.free(t)
        return out, [int(lens[p]) for p in parents], pairs

    def compact(self, tables: Sequence[Sequence[int]]) -> Tuple[List[List[int]], List[Tuple[int, int]]]:
        """Moves the pages in use to the front: with ``n`` pages in use, those beyond page ``n`` go to the free
        ones before it.  ``tables``: those of all requests.  Returns the new tables and the ``(from, to)`` pairs; targets are free pages, so
        never sources."""
        used = np.flatnonzero(self.uses > 0)
        n = len(used)
        high = used[used >= n]
        low = np.flatnonzero(self.uses[:n] == 0)
        self.uses[low], self.uses[high] = self.uses[high], 0
        to = np.arange(self.num_pages)
        to[high] = low
        moved = [to[np.asarray(t, dtype=np.int64)].tolist() if len(t) else [] for t in tables]
        return moved, list(zip(high.tolist(), low.tolist()))
