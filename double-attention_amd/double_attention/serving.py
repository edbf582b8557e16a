"""Sequences that a ``DoubleAttentionLM`` continues over paged caches.

``CachedSequences`` keeps what the operators of ``serving_ops`` leave to the
program: which pages are whose and which are free, the lengths and positions,
and the weights that cached tokens gathered.
"""

from __future__ import annotations

from typing import Iterator, Sequence

import torch
from torch import Tensor

from .modules import DoubleAttentionLM
from .serving_ops import PagedCache, cache_compact_hip, cache_select_hip


class CachedSequences:
    """A number of sequences of one model, in one pool of pages.

    ``pages`` pages of ``page_size`` tokens hold every layer's routed keys and
    values; a sequence takes pages as it grows, up to the model's
    ``max_sequence_length`` positions.  With ``gather_weights`` every cached
    token's attention is gathered, and ``evict`` cuts sequences to the tokens
    that got most of it; their positions go on as if nothing had been cut.

    Lengths and pages are kept on the host; nothing is read back from the
    device (its small tables are copied there in each call, which waits for what
    the stream still does).  A call that raises changes nothing: pages, lengths
    and gathered weights (of which there are two buffers) are the new ones when
    all of its work has been enqueued.  Use one stream: pages that were freed are
    written anew by later calls.
    """

    def __init__(
        self, model: DoubleAttentionLM, sequences: int, pages: int, *, page_size: int = 64, gather_weights: bool = False
    ) -> None:
        if sequences < 1:
            raise ValueError("CachedSequences: needs at least one sequence")
        self.model = model
        self.caches = model.paged_caches(pages, page_size)
        self.page_size = page_size
        self.entries = min(pages, -(-model.max_sequence_length // page_size))
        self.lengths = [0] * sequences     # cached tokens
        self.positions = [0] * sequences   # of the next token
        self._pages: list[list[int]] = [[] for _ in range(sequences)]
        self._free = list(range(pages - 1, -1, -1))
        self._device = self.caches[0].keys.device
        self.weights = self._next_weights = None
        if gather_weights:
            self.weights = torch.zeros(
                len(self.caches), sequences, self.entries * page_size, dtype=torch.float32, device=self._device
            )
            self._next_weights = torch.empty_like(self.weights)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages(self, sequence: int) -> Tensor:
        """A sequence's pages in order (for ``PagedCache.rows``)."""

        return torch.tensor(self._pages[sequence], dtype=torch.int64, device=self._device)

    def _table(self, pages: Sequence[Sequence[int]]) -> Tensor:
        rows = [[*row, *[-1] * (self.entries - len(row))] for row in pages]
        return torch.tensor(rows, dtype=torch.int32).to(self._device)

    def _count(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def _last_free(self, pages: int) -> Iterator[int]:
        return reversed(self._free[len(self._free) - pages:])

    def extend(self, token_ids: Tensor, counts: Sequence[int], *, last_only: bool = False) -> Tensor:
        """Continues sequence b by ``counts[b]`` tokens (0: not at all).

        ``token_ids``: int64 ``[sum(counts)]``, the sequences' new tokens one
        after the other (ids on the host are checked against the vocabulary).
        Returns the logits of all of them, or with ``last_only`` of each
        continued sequence's last one, in order.
        """

        counts = [int(n) for n in counts]
        if len(counts) != len(self.lengths) or min(counts) < 0:
            raise ValueError(f"extend: counts are {len(self.lengths)} numbers of new tokens, got {counts}")
        total = sum(counts)
        if token_ids.dtype is not torch.int64 or token_ids.shape != (total,):
            raise ValueError(f"extend: token_ids are int64 [{total}], got {token_ids.dtype} {tuple(token_ids.shape)}")
        limit, vocab = self.model.max_sequence_length, self.model.token_embedding.num_embeddings
        for b, n in enumerate(counts):
            if self.positions[b] + n > limit:
                raise ValueError(f"extend: sequence {b} would end at {self.positions[b] + n} tokens; the model has {limit} positions")
        if token_ids.device.type == "cpu" and total and not 0 <= int(token_ids.min()) <= int(token_ids.max()) < vocab:
            raise ValueError(f"extend: token_ids must be in [0, {vocab})")
        lengths = [length + n for length, n in zip(self.lengths, counts)]
        need = [self._count(length) - len(own) for length, own in zip(lengths, self._pages)]
        for b, own in enumerate(self._pages):
            if len(own) + need[b] > self.entries:
                raise RuntimeError(f"extend: sequence {b} does not fit {self.entries} pages")
        if sum(need) > len(self._free):
            raise RuntimeError(f"extend: needs {sum(need)} more pages, {len(self._free)} are free")
        taken = self._last_free(sum(need))
        pages = [[*own, *(next(taken) for _ in range(n))] if n else own for own, n in zip(self._pages, need)]
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        positions = [p for at, n in zip(self.positions, counts) for p in range(at, at + n)]
        sequences = len(counts)
        numbers = torch.tensor(lengths + offsets, dtype=torch.int32).to(self._device)
        last = [end - 1 for end, n in zip(offsets[1:], counts) if n]
        logits = self.model.cached_forward(
            token_ids.to(self._device), torch.tensor(positions, dtype=torch.int64).to(self._device), self.caches,
            self._table(pages), numbers[:sequences], numbers[sequences:], weights=self.weights, weights_out=self._next_weights,
            rows=torch.tensor(last, dtype=torch.int64).to(self._device) if last_only else None,
            max_chunk=max(1, *counts), max_length=max(1, *lengths),
        )
        # Nothing below raises.
        del self._free[len(self._free) - sum(need):]
        self._pages, self.lengths = pages, lengths
        self.positions = [at + n for at, n in zip(self.positions, counts)]
        self.weights, self._next_weights = self._next_weights, self.weights
        return logits

    @torch.inference_mode()   # the tensors may have been made there
    def evict(self, keep: int, recent: int = 0) -> None:
        """Cuts every sequence of more than ``keep`` tokens, in each layer by itself,
        to its last ``recent`` tokens and those of the others that gathered the
        largest weights.  The kept tokens move into free pages, of as many
        sequences at a time as those take, whose own pages become free; where
        none are left for one sequence, through temporary memory."""

        if self.weights is None:
            raise RuntimeError("evict: the sequences were made without gather_weights")
        if keep < 1 or not 0 <= recent <= keep:
            raise ValueError(f"evict: needs 1 <= keep and 0 <= recent <= keep, got {keep} and {recent}")
        cut = [b for b, length in enumerate(self.lengths) if length > keep]
        if not cut:
            return
        each = self._count(keep)
        # The rounds' page tables: before, after, and of the temporary pages.  Pages
        # of the sequences that stay in a round are not named: nothing of theirs moves.
        pages, free, rounds = list(self._pages), list(self._free), []
        waiting = cut
        while waiting:
            fit = len(free) // each
            group, waiting = waiting[:max(1, fit)], waiting[max(1, fit):]
            after: list[list[int]] = [[] for _ in pages]
            for b in group:
                after[b] = [free.pop() for _ in range(each)] if fit else pages[b][:each]
            through = None if fit else self._table([list(range(len(row))) for row in after])
            rounds.append((self._table(pages), self._table(after), through))
            for b in group:
                free.extend(reversed(pages[b] if fit else pages[b][each:]))
                pages[b] = after[b]
        lengths = torch.tensor(self.lengths, dtype=torch.int32).to(self._device)
        chosen = [cache_select_hip(weights, lengths, keep, recent) for weights in self.weights]
        if any(through is not None for *_, through in rounds):
            temporary = [PagedCache(*(t.new_empty(each, *t.shape[1:]) for t in cache)) for cache in self.caches]
            in_order = torch.arange(keep, dtype=torch.int32, device=self._device).repeat(len(pages), 1)
        for n, (table, new_table, through) in enumerate(rounds):
            for layer, (cache, (kept, counts)) in enumerate(zip(self.caches, chosen)):
                out, to = (cache, new_table) if through is None else (temporary[layer], through)
                if n == 0:   # the last that needs memory; no page of a sequence has been written yet
                    moved = cache_compact_hip(cache, table, kept, counts, out, to, weights=self.weights[layer])
                    self._next_weights[layer].copy_(moved)
                else:
                    cache_compact_hip(cache, table, kept, counts, out, to)
            if through is not None:
                for cache, held, (_, counts) in zip(self.caches, temporary, chosen):
                    cache_compact_hip(held, through, in_order, counts, cache, new_table)
        self._pages, self._free = pages, free
        for b in cut:
            self.lengths[b] = keep
        self.weights, self._next_weights = self._next_weights, self.weights

    def release(self, sequence: int) -> None:
        """Frees a sequence's pages; it starts anew, empty."""

        self._free.extend(reversed(self._pages[sequence]))
        self._pages[sequence] = []
        self.lengths[sequence] = self.positions[sequence] = 0


__all__ = ["CachedSequences"]
