"""``CachedSequences`` around calls that raise and pools without a free page."""

from __future__ import annotations

import pytest
import torch

import double_attention as da
from double_attention import serving
from test_serving_model import ids, model_of


def state_of(s: da.CachedSequences):
    weights = None if s.weights is None else s.weights.clone()
    return [list(p) for p in s._pages], list(s._free), list(s.lengths), list(s.positions), weights


def same(a, b) -> bool:
    return a[:4] == b[:4] and ((a[4] is None and b[4] is None) or torch.equal(a[4], b[4]))


class Failure(RuntimeError):
    pass


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch) -> None:
    monkeypatch.setattr(da.DoubleAttentionLM, "_cached_dtype", lambda model: model.token_embedding.weight.dtype)


class Forward:
    """Stands in for ``cached_forward`` on the host: adds one to the weights of every
    cached token, layer by layer, and fails in layer ``fails``."""

    def __init__(self, model, fails=None) -> None:
        self.model, self.fails = model, fails

    def __call__(self, token_ids, positions, caches, table, lengths, offsets, *, weights=None, weights_out=None, rows=None, **hints):
        for layer in range(len(caches)):
            if layer == self.fails:
                raise Failure("out of memory")
            if weights is not None:
                there = torch.arange(weights.shape[2])[None] < lengths[:, None]
                (weights if weights_out is None else weights_out)[layer] = torch.where(there, weights[layer] + 1, 0.0)
        return torch.zeros(len(token_ids) if rows is None else len(rows), 97)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("fails", [0, 1])
def test_a_forward_that_raises_changes_nothing(gather, fails, monkeypatch) -> None:
    model = model_of()
    s = da.CachedSequences(model, 3, 7, page_size=32, gather_weights=gather)
    monkeypatch.setattr(model, "cached_forward", Forward(model))
    s.extend(torch.cat(ids(40, 5, 0)), [40, 5, 0])
    before = state_of(s)
    monkeypatch.setattr(model, "cached_forward", Forward(model, fails))
    for counts in ([50, 0, 10], [1, 1, 1], [0, 0, 96]):
        with pytest.raises(Failure):
            s.extend(torch.cat(ids(*counts)), counts)
        assert same(state_of(s), before)
    # What the others lack is not hidden by pages that a failed call had taken.
    with pytest.raises(RuntimeError, match="needs 6 more pages, 4 are free"):
        s.extend(torch.cat(ids(0, 92, 96)), [0, 92, 96])
    assert same(state_of(s), before)
    monkeypatch.setattr(model, "cached_forward", Forward(model))
    s.extend(torch.cat(ids(50, 0, 10)), [50, 0, 10])
    assert s.lengths == [90, 5, 10] and s.positions == [90, 5, 10] and s.free_pages == 2
    assert sorted(sum(s._pages, s._free)) == list(range(7))
    if gather:
        # Two forwards counted each of the first tokens, one the others.
        for b, (old, new) in enumerate(((40, 90), (5, 5), (0, 10))):
            expected = torch.zeros(s.weights.shape[2])
            expected[:new] = 1
            expected[:old] = 2
            assert torch.equal(s.weights[0, b], expected) and torch.equal(s.weights[1, b], expected)


def plain_select(weights, lengths, keep, recent):
    kept = torch.full((len(lengths), keep), -1, dtype=torch.int32)
    counts = lengths.clamp(max=keep)
    for b, n in enumerate(lengths.tolist()):
        count = min(n, keep)
        r = min(recent, count)
        heavy = torch.sort(weights[b, :n - r], descending=True, stable=True).indices[:count - r]
        kept[b, :count] = torch.cat((heavy.sort().values, torch.arange(n - r, n))).int()
    return kept, counts


def plain_compact(cache, table, kept, counts, out, out_table, *, weights=None):
    moved = None if weights is None else torch.zeros(len(kept), out_table.shape[1] * out.page_size)
    for b, count in enumerate(counts.tolist()):
        for i, t in enumerate(kept[b, :count].tolist()):
            if weights is not None:
                moved[b, i] = weights[b, t]
            to, at = int(out_table[b, i // out.page_size]), int(table[b, t // cache.page_size])
            if to >= 0 and at >= 0:
                out.keys[to, i % out.page_size] = cache.keys[at, t % cache.page_size]
                out.values[to, i % out.page_size // 32, :, i % 32] = cache.values[at, t % cache.page_size // 32, :, t % 32]
    return moved


def filled(sequences, pages, counts, monkeypatch, gather=True):
    """Sequences on the host with random cached rows, whose moves are plain ones."""

    model = model_of()
    s = da.CachedSequences(model, sequences, pages, page_size=32, gather_weights=gather)
    monkeypatch.setattr(model, "cached_forward", Forward(model))
    monkeypatch.setattr(serving, "cache_select_hip", plain_select)
    monkeypatch.setattr(serving, "cache_compact_hip", plain_compact)
    s.extend(torch.cat(ids(*counts)), counts)
    g = torch.Generator().manual_seed(1)
    for cache in s.caches:
        cache.keys.copy_(torch.randn(cache.keys.shape, generator=g))
        cache.values.copy_(torch.randn(cache.values.shape, generator=g))
    for b, n in enumerate(counts):
        s.weights[:, b, :n] = torch.rand(len(s.caches), n, generator=g)
    return s


@pytest.mark.parametrize("pages", [14, 8])
@pytest.mark.parametrize("fails", [0, 1, 2, 3])
def test_an_eviction_that_raises_changes_nothing(fails, pages, monkeypatch) -> None:
    s = filled(3, pages, [100, 20, 70], monkeypatch)
    before = state_of(s)
    rows = [[[t.clone() for t in c.rows(s.pages(b), n)] for b, n in enumerate(s.lengths)] for c in s.caches]
    calls = iter(range(100))

    def failing(call):
        def run(*args, **kwargs):
            if next(calls) == fails:
                raise Failure("out of memory")
            return call(*args, **kwargs)

        return run

    with monkeypatch.context() as m:
        m.setattr(serving, "cache_select_hip", failing(plain_select))
        m.setattr(serving, "cache_compact_hip", failing(plain_compact))
        with pytest.raises(Failure):
            s.evict(40, 8)
    assert same(state_of(s), before)
    for cache, of_layer in zip(s.caches, rows):
        for b, n in enumerate(s.lengths):
            assert all(torch.equal(*pair) for pair in zip(cache.rows(s.pages(b), n), of_layer[b]))
    s.evict(40, 8)
    assert s.lengths == [40, 20, 40] and sorted(sum(s._pages, s._free)) == list(range(pages))


def test_refusals_of_a_second_buffer_of_weights() -> None:
    model = model_of()
    token, ends = torch.zeros(1, dtype=torch.int64), torch.tensor([0, 1], dtype=torch.int32)
    where = (token, token, model.paged_caches(2, 32), torch.zeros(1, 1, dtype=torch.int32), ends[1:], ends)
    weights = torch.zeros(2, 1, 32)
    both = torch.zeros(3, 1, 32)
    for first, second in ((None, weights), (weights, weights[:1]), (weights, torch.zeros(2, 1, 64)[..., ::2]), (both[:2], both[1:]),
                          (both[1:], both[:2])):
        with pytest.raises(ValueError, match="weights_out"):
            model.cached_forward(*where, weights=first, weights_out=second)


@pytest.mark.gpu
def test_a_failed_forward_can_be_made_again(monkeypatch) -> None:
    model = model_of("two-maps").cuda()
    counts, chunk = [40, 70], torch.cat(ids(3, 30, seed=1))
    s, other = (da.CachedSequences(model, 2, 8, page_size=32, gather_weights=True) for _ in range(2))
    for t in (s, other):
        t.extend(torch.cat(ids(*counts)), counts)
    before = state_of(s)

    def failing(*args):
        raise Failure("out of memory")

    with monkeypatch.context() as m:
        m.setattr(model.stack.blocks[1], "_hip_cached_block", failing)
        with pytest.raises(Failure):
            s.extend(chunk, [3, 30])
    assert same(state_of(s), before)
    assert torch.equal(s.extend(chunk, [3, 30]), other.extend(chunk, [3, 30]))
    assert same(state_of(s), state_of(other))
    weights = s.weights.clone()
    s.extend(chunk[:0], [0, 0])   # no new token: nothing gathered
    assert torch.equal(s.weights, weights)


def check_eviction(s, keep, recent, select) -> None:
    """The pages hold what ``select`` chose before, and every page has one owner."""

    lengths, pages = list(s.lengths), len(sum(s._pages, s._free))
    rows = [[[t.clone() for t in c.rows(s.pages(b), n)] for b, n in enumerate(lengths)] for c in s.caches]
    weights = s.weights.clone()
    on_device = torch.tensor(lengths, dtype=torch.int32, device=weights.device)
    chosen = [select(w.contiguous(), on_device, keep, recent) for w in weights]
    positions = list(s.positions)
    s.evict(keep, recent)
    assert s.lengths == [min(n, keep) for n in lengths] and s.positions == positions
    assert sorted(sum(s._pages, s._free)) == list(range(pages))
    assert [len(p) for p in s._pages] == [-(-n // s.page_size) for n in s.lengths]
    for layer, cache in enumerate(s.caches):
        kept, counts = chosen[layer]
        for b, n in enumerate(s.lengths):
            assert int(counts[b]) == n
            stays = kept[b, :n].long()
            got = cache.rows(s.pages(b), n)
            assert all(torch.equal(t, before[stays]) for t, before in zip(got, rows[layer][b]))
            expected = torch.zeros_like(weights[layer, b])
            expected[:n] = weights[layer, b][stays]
            assert torch.equal(s.weights[layer, b], expected)


# 12 pages for sequences of 4, 1, 3 and 4 pages, cut to two pages each: none free,
# one too few for a sequence, for two and for all at once; and a page that a cut
# sequence keeps all of.
@pytest.mark.parametrize("pages,keep,recent", [(12, 40, 8), (13, 40, 8), (14, 40, 0), (17, 40, 40), (20, 40, 8), (12, 96, 3), (12, 64, 1),
                                               (12, 1, 0), (13, 33, 2), (12, 127, 0)])
def test_pools_without_room_are_cut(pages, keep, recent, monkeypatch) -> None:
    check_eviction(filled(4, pages, [100, 20, 70, 128], monkeypatch), keep, recent, plain_select)


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [12, 13, 16])
def test_pools_without_room_are_cut_on_the_device(pages) -> None:
    model = model_of("two-maps").cuda()
    s = da.CachedSequences(model, 4, pages, page_size=32, gather_weights=True)
    s.extend(torch.cat(ids(100, 20, 70, 127)), [100, 20, 70, 127])
    s.extend(torch.cat(ids(0, 1, 0, 1, seed=1)), [0, 1, 0, 1])
    check_eviction(s, 40, 8, da.cache_select_hip)
    other = da.CachedSequences(model, 4, pages, page_size=32, gather_weights=True)
    other._pages, other._free = [list(p) for p in s._pages], list(s._free)
    other.lengths, other.positions, other.weights = list(s.lengths), list(s.positions), s.weights.clone()
    for mine, theirs in zip(other.caches, s.caches):
        mine.keys.copy_(theirs.keys)
        mine.values.copy_(theirs.values)
    # What was left behind in the pages reaches nothing.
    for cache in other.caches:
        for p in other._free:
            cache.keys[p] = float("nan")
            cache.values[p] = float("nan")
    tokens = torch.cat(ids(3, 1, 0, 2, seed=2))
    assert torch.equal(s.extend(tokens, [3, 1, 0, 2]), other.extend(tokens, [3, 1, 0, 2]))
