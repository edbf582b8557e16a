"""The serving operators against plain 64-bit forms.

Tolerances count roundings: half a step of the 16-bit type
(``torch.finfo(t).eps / 2`` of the value) for what is rounded to it, 2^-24 for
each fp32 operation, bounded term by term beside each test.
"""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

import double_attention as da
from double_attention import _lib, serving_ops

F32 = 2.0 ** -24   # half a step of fp32
TYPES = [(torch.float16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)]


def _device() -> torch.device:
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    if not da.HIP_AVAILABLE:
        raise RuntimeError("HIP library not built; run python double-attention_amd/build.py")
    return torch.device("cuda")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, expected, tolerance):
    assert got.shape == expected.shape
    nan, same = torch.isnan(expected), got.double() == expected   # infinities have no difference
    assert torch.equal(torch.isnan(got), nan)
    off = (got.double() - expected).abs()[~nan & ~same]
    worst = (off - tolerance.expand_as(expected)[~nan & ~same]).max().item() if off.numel() else 0.0
    assert worst <= 0, f"off by {off.max().item():.3e}, {worst:.3e} more than allowed"


class Setup:
    """Sequences in a pool whose unused slots hold NaN, and their new tokens."""

    def __init__(self, lengths, chunks, branches=1, routing_dim=64, value_dim=64, page=32, types=TYPES[0], seed=0, spare=2,
                 front=0, behind=0, spread=1.0):
        device = _device()
        g = torch.Generator().manual_seed(seed)
        self.lengths_list, self.chunks = lengths, chunks
        self.page, self.branches, self.routing_dim, self.value_dim = page, branches, routing_dim, value_dim
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=g).tolist()
        entries = max(counts + [1])
        table = torch.full((len(lengths), entries), -1, dtype=torch.int32)
        keys = torch.full((pages, page, branches, routing_dim), math.nan)
        values = torch.full((pages, page // 32, value_dim, 32), math.nan)
        self.rows = []
        for b, (n, count) in enumerate(zip(lengths, counts)):
            mine = [order.pop() for _ in range(count)]
            table[b, :count] = torch.tensor(mine, dtype=torch.int32)
            k = torch.nn.functional.normalize(torch.randn(n, branches, routing_dim, generator=g), dim=-1) * spread
            v = torch.randn(n, value_dim, generator=g)
            k, v = k.to(types[0]), v.to(types[1])
            self.rows.append((k.double(), v.double()))
            for t in range(n):
                keys[mine[t // page], t % page] = k[t].float()
                values[mine[t // page], t % page // 32, :, t % 32] = v[t].float()
        offsets = [front]
        for n in chunks:
            offsets.append(offsets[-1] + n)
        total = offsets[-1] + behind
        q = torch.nn.functional.normalize(torch.randn(total, branches, routing_dim, generator=g), dim=-1) * spread
        self.query = q.to(types[0]).to(device)
        self.cache = da.PagedCache(keys.to(types[0]).to(device), values.to(types[1]).to(device))
        self.table, self.lengths = table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)
        self.offsets = torch.tensor(offsets, dtype=torch.int32, device=device)
        self.types, self.total, self.front, self.spread = types, total, front, spread

    def where(self):
        return self.query, self.cache, self.table, self.lengths, self.offsets

    def exact(self, scales, causal=True, mix=None, dropped=()):
        """``(out, tolerance, weights, tolerance of the weights)``; tokens of the
        (sequence, page entry) pairs in ``dropped`` are not there."""

        maps = len(scales)
        out = torch.zeros(self.total, maps, self.value_dim, dtype=torch.float64)
        size = torch.zeros_like(out)
        capacity = self.table.shape[1] * self.page
        weights = torch.zeros(len(self.chunks), capacity, dtype=torch.float64)
        group = max(1, self.branches // maps)
        start = self.front
        longest = 0
        for b, (n, new) in enumerate(zip(self.lengths_list, self.chunks)):
            k, v = self.rows[b]
            q = self.query[start:start + new].double().cpu()
            positions = torch.arange(n - new, n)
            seen = torch.arange(n)[None] <= positions[:, None] if causal else torch.ones(new, n, dtype=torch.bool)
            for entry in (e for s, e in dropped if s == b):
                seen[:, entry * self.page:(entry + 1) * self.page] = False
            longest = max(longest, n)
            for s in range(maps):
                h = range(s * group, (s + 1) * group) if self.branches >= maps else [s // (maps // self.branches)]
                scores = sum(q[:, i] @ k[:, i].T for i in h) * float(scales[s]) / math.sqrt(len(h))
                scores = scores.masked_fill(~seen, -math.inf)
                empty = ~seen.any(1)
                p = torch.softmax(scores.masked_fill(empty[:, None], 0.0), -1) * ~empty[:, None]
                out[start:start + new, s] = p @ v
                size[start:start + new, s] = p @ v.abs()
                weights[b, :n] += p.sum(0)
            start += new
        # A score is off by its sum of fp32 products (each partial sum at most
        # the product of the rows' lengths) and the product with the scale, its
        # exponent by the difference to the maximum (at most twice the score) and
        # the exponential itself by two steps.
        width = group * self.routing_dim
        length = self.spread ** 2 * group * 1.02
        top = float(scales.abs().max())
        delta = top * length * (width + 8) * F32 + 8 * F32
        half = half_step(self.types[1])
        # Probabilities are rounded once (in fp16 by 2^-25 at least, beside a sum
        # of at least 1/2: the reference is the maximum rounded up to a whole
        # number); numerator and denominator carry the scores' errors.  No value
        # exceeds 6.
        tolerance = (half + 2 * delta + 16 * F32) * size + half * out.abs()
        if self.types[1] is torch.float16:
            tolerance = tolerance + longest * 2.0 ** -25 * 2 * 6.0
        tolerance = tolerance + 2.0 ** -25
        if mix is not None:
            m = mix.double().cpu()[None, :, None]
            out, tolerance = (out * m).sum(1), ((tolerance + 4 * F32 * size) * m.abs()).sum(1) + half * (out * m).sum(1).abs()
        rows = max(self.chunks + [1]) * maps
        return out, tolerance, weights, weights * (2 * delta + (rows + 8) * F32) + 1e-30


def scales_of(maps, top=16.0):
    return torch.linspace(1.0, 0.6, maps) * top


CASES = [
    # lengths, chunks, (branches, maps, routing_dim), value_dim, page
    pytest.param([1], [1], (1, 1, 64), 64, 32, id="one-token"),
    pytest.param([33], [1], (1, 1, 256), 512, 32, id="page-end"),
    pytest.param([31, 32, 33, 64, 65, 1, 500], [1] * 7, (1, 1, 256), 512, 64, id="decode-edges"),
    pytest.param([5, 40, 0, 129], [5, 7, 0, 129], (1, 1, 128), 192, 32, id="ragged-empty"),
    pytest.param([70, 300, 17], [16, 17, 1], (2, 2, 64), 320, 96, id="two-maps"),
    pytest.param([100, 64], [31, 33], (4, 4, 128), 512, 128, id="four-maps"),
    pytest.param([90, 20], [4, 3], (2, 1, 256), 256, 64, id="grouped"),
    pytest.param([90, 211], [40, 3], (1, 2, 256), 128, 64, id="repeated"),
    pytest.param([50, 77], [2, 50], (1, 1, 512), 1024, 32, id="wide"),
    pytest.param([50, 77], [2, 50], (1, 1, 64), 64, 32, id="narrow"),
    pytest.param([1000, 3], [130, 3], (1, 3, 64), 576, 32, id="three-maps-odd-width"),
    pytest.param([700], [300], (1, 1, 256), 512, 64, id="chunk"),
    pytest.param([2100, 260, 90], [257, 260, 1], (1, 1, 256), 512, 64, id="chunks-and-token"),
    pytest.param([9000], [1], (1, 1, 64), 64, 64, id="long"),
    pytest.param([3000, 40, 700], [2, 40, 1], (4, 2, 192), 384, 160, id="keys-of-768"),
    pytest.param([500, 130], [9, 1], (2, 2, 512), 768, 32, id="keys-of-1024"),
    pytest.param([500, 130], [9, 1], (2, 1, 256), 2112, 32, id="five-slices"),
    pytest.param([130, 300], [1, 7], (1, 1, 320), 192, 32, id="keys-of-320"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lengths,chunks,layout,value_dim,page", CASES)
def test_paged_attention(lengths, chunks, layout, value_dim, page, types, causal) -> None:
    branches, maps, routing_dim = layout
    s = Setup(lengths, chunks, branches, routing_dim, value_dim, page, types)
    scales = scales_of(maps)
    expected, tolerance, weights, w_tolerance = s.exact(scales, causal)
    got = da.paged_attention_hip(*s.where(), scales.to(s.query.device), causal)
    close(got.cpu(), expected, tolerance)
    hinted, gathered = da.paged_attention_weights_hip(*s.where(), scales.to(s.query.device), causal, max_chunk=max(chunks),
                                                      max_length=max(lengths))
    close(hinted.cpu(), expected, tolerance)
    close(gathered.cpu(), weights, w_tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("maps", [1, 2, 4])
def test_paged_attention_mix_and_other_rows(types, maps) -> None:
    s = Setup([77, 300, 64, 1], [9, 1, 64, 1], maps, 64, 192, 64, types, front=3, behind=40)
    scales = scales_of(maps)
    mix = torch.softmax(torch.arange(maps, dtype=torch.float32), 0)
    expected, tolerance, _, _ = s.exact(scales, True, mix)
    got = da.paged_attention_hip(*s.where(), scales.to(s.query.device), mix=mix.to(s.query.device))
    close(got.cpu(), expected, tolerance)
    assert not got[:3].any() and not got[-40:].any()
    expected, tolerance, _, _ = s.exact(scales, True)
    got = da.paged_attention_hip(*s.where(), scales.to(s.query.device), max_length=1)
    close(got.cpu(), expected, tolerance)
    assert not got[:3].any() and not got[-40:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [[1, 1, 1], [20, 40, 1], [150, 2, 200]])
def test_paged_attention_any_hint(chunks) -> None:
    """The hints choose the launch, not the result."""

    s = Setup([200, 90, 333], chunks, 1, 128, 256, 32)
    scales = scales_of(1)
    expected, tolerance, weights, w_tolerance = s.exact(scales)
    for max_chunk, max_length in ((1, 1), (1, None), (33, 100), (4096, 100000)):
        got, gathered = da.paged_attention_weights_hip(*s.where(), scales.cuda(), max_chunk=max_chunk, max_length=max_length)
        close(got.cpu(), expected, tolerance)
        close(gathered.cpu(), weights, w_tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [[1, 1], [70, 130]])
@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31)])
def test_paged_attention_pages_that_are_not_there(bad, chunks) -> None:
    s = Setup([200, 333], chunks, 1, 64, 128, 32)
    s.table[0, 2] = bad
    s.table[1, 0] = bad
    s.table[1, 10] = bad   # with the newest tokens in it
    scales = scales_of(1)
    expected, tolerance, weights, w_tolerance = s.exact(scales, dropped=[(0, 2), (1, 0), (1, 10)])
    got, gathered = da.paged_attention_weights_hip(*s.where(), scales.cuda())
    close(got.cpu(), expected, tolerance)
    close(gathered.cpu(), weights, w_tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [[3, 1], [100, 70]])
def test_paged_attention_lengths_that_do_not_fit(chunks) -> None:
    """More new tokens than tokens: those in front of the sequence see nothing.
    Lengths behind the table: what it has is seen."""

    s = Setup([96, 128], chunks, 1, 64, 128, 32)
    out = da.paged_attention_hip(*s.where(), scales_of(1).cuda())
    s.lengths[0] = 2
    got, gathered = da.paged_attention_weights_hip(*s.where(), scales_of(1).cuda())
    front = chunks[0] - 2
    assert front >= 1 and not got[:front].any() and bool(got[front].any()) and not got.isnan().any()
    assert gathered[0, 2:].sum() == 0
    # Its first token sees itself alone.
    assert torch.equal(got[front, 0].double().cpu(), s.rows[0][1][0])
    close(got[chunks[0]:].cpu(), out[chunks[0]:].double().cpu(), torch.zeros(1, dtype=torch.float64))
    s.lengths[1] = 1 << 30
    got = da.paged_attention_hip(*s.where(), scales_of(1).cuda())   # every new token stands behind all that are there
    k, v = s.rows[1]
    q = s.query[chunks[0]:].double().cpu()[:, 0]
    p = torch.softmax(16.0 * q @ k[:, 0].T, -1)
    delta = 16.0 * 1.02 * 72 * F32 + 8 * F32
    half = half_step(torch.bfloat16)
    close(got[chunks[0]:, 0].cpu(), p @ v, (half + 2 * delta + 16 * F32) * (p @ v.abs()) + half * (p @ v).abs())
    s.lengths[:] = -5
    assert not da.paged_attention_hip(*s.where(), scales_of(1).cuda()).any()


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 50, 200])
def test_paged_attention_extreme_scores(chunk) -> None:
    """Sharp and flat distributions, negative and zero scales."""

    for top in (1000.0, 0.0, -16.0, 1e-6):
        s = Setup([300], [chunk], 1, 64, 64, 32, TYPES[2], seed=3)
        scales = torch.tensor([top])
        expected, tolerance, weights, w_tolerance = s.exact(scales)
        got, gathered = da.paged_attention_weights_hip(*s.where(), scales.cuda())
        close(got.cpu(), expected, tolerance)
        close(gathered.cpu(), weights, w_tolerance + 1e-9)


@pytest.mark.gpu
@pytest.mark.parametrize("chunks", [[1, 1], [150, 3]])
def test_paged_attention_views(chunks) -> None:
    """A layer's pages out of a tensor of several layers, queries out of routed
    pairs, a table with a wider pitch, 16-bit scales."""

    s = Setup([200, 333], chunks, 2, 64, 128, 32)
    layers = torch.full((s.cache.keys.shape[0], 3, *s.cache.keys.shape[1:]), math.nan, dtype=torch.float16, device="cuda")
    layers[:, 1] = s.cache.keys
    v_layers = torch.full((s.cache.values.shape[0], 2, *s.cache.values.shape[1:]), math.nan, dtype=torch.bfloat16, device="cuda")
    v_layers[:, 0] = s.cache.values
    pairs = torch.stack((s.query, torch.full_like(s.query, math.nan)), 1)
    wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, :s.table.shape[1]] = s.table
    scales = scales_of(2).half()
    expected, tolerance, _, _ = s.exact(scales)
    view = da.PagedCache(layers[:, 1], v_layers[:, 0])
    got = da.paged_attention_hip(pairs[:, 0], view, wide[:, :s.table.shape[1]], s.lengths, s.offsets, scales.cuda())
    close(got.cpu(), expected, tolerance)
    odd = torch.empty(s.query.numel() + 1, dtype=torch.float16, device="cuda")[1:].view_as(s.query).copy_(s.query)
    again = da.paged_attention_hip(odd.transpose(1, 2).contiguous().transpose(1, 2), view, wide, s.lengths, s.offsets, scales.cuda())
    close(again.cpu(), expected, tolerance)   # a wider table: other parts


@pytest.mark.gpu
def test_paged_weights_accumulate_in_place() -> None:
    s = Setup([200, 90, 333], [5, 1, 40], 2, 64, 64, 32)
    scales = scales_of(2)
    _, _, added, tolerance = s.exact(scales)
    before = torch.rand(3, s.table.shape[1] * 32, generator=torch.Generator().manual_seed(1)) + 0.5
    old = torch.arange(before.shape[1])[None] < torch.tensor([195, 89, 293])[:, None]
    expected = torch.where(old, before.double(), 0.0) + added
    _, fresh = da.paged_attention_weights_hip(*s.where(), scales.cuda(), weights=before.cuda())
    close(fresh.cpu(), expected, tolerance + F32 * 2 * expected)
    held = before.cuda()
    _, same = da.paged_attention_weights_hip(*s.where(), scales.cuda(), weights=held, out=held)
    assert same is held and torch.equal(held, fresh)
    # No new rows at all: the weights are what they were.
    none = torch.zeros(4, dtype=torch.int32, device="cuda")
    out, same = da.paged_attention_weights_hip(s.query[:0], s.cache, s.table, s.lengths, none, scales.cuda(), weights=before.cuda())
    inside = torch.arange(before.shape[1])[None] < torch.tensor([200, 90, 333])[:, None]
    assert out.shape == (0, 2, 64) and torch.equal(same.cpu(), torch.where(inside, before, 0.0))


@pytest.mark.gpu
def test_paged_attention_is_the_modules_attention() -> None:
    """A whole prompt as one chunk is what ``routed_attention_hip`` gives."""

    s = Setup([300, 300], [300, 300], 2, 128, 256, 64)
    scales = scales_of(2)
    got = da.paged_attention_hip(*s.where(), scales.cuda())
    k = torch.stack([r[0] for r in s.rows]).half().cuda()
    v = torch.stack([r[1] for r in s.rows]).bfloat16().cuda()
    other = da.routed_attention_hip(s.query.view(2, 300, 2, 128).transpose(1, 2), k.transpose(1, 2), v, scales.cuda())
    expected, tolerance, _, _ = s.exact(scales)
    close(got.cpu(), expected, tolerance)
    # Both are within their tolerance of the definition.
    close(got.cpu(), other.transpose(1, 2).reshape(600, 2, 256).double().cpu(), 2 * tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lengths,chunks,branches,routing_dim,value_dim,page", [
    ([1], [1], 1, 64, 64, 32),
    ([33, 32, 31, 64, 300, 7], [1, 1, 1, 1, 1, 1], 1, 256, 512, 64),
    ([40, 0, 129, 200], [40, 0, 70, 33], 2, 64, 192, 96),
    ([777, 100], [700, 65], 4, 128, 576, 128),
])
def test_cache_append(lengths, chunks, branches, routing_dim, value_dim, page, types) -> None:
    s = Setup(lengths, chunks, branches, routing_dim, value_dim, page, types, front=2, behind=3)
    key, value = torch.full_like(s.query, 7.0), torch.full((s.total, value_dim), 7.0, dtype=types[1], device="cuda")
    for b, new in enumerate(chunks):
        at = int(s.offsets[b])
        if new:
            key[at:at + new] = s.rows[b][0][-new:].to(types[0]).cuda()
            value[at:at + new] = s.rows[b][1][-new:].to(types[1]).cuda()
    empty = da.PagedCache(torch.full_like(s.cache.keys, 3.0), torch.full_like(s.cache.values, 3.0))
    expected_k, expected_v = empty.keys.clone(), empty.values.clone()
    for b, (n, new) in enumerate(zip(lengths, chunks)):
        for t in range(n - new, n):
            at = int(s.table[b, t // page])
            expected_k[at, t % page] = s.rows[b][0][t].to(types[0]).cuda()
            expected_v[at, t % page // 32, :, t % 32] = s.rows[b][1][t].to(types[1]).cuda()
    for hint in (None, max(chunks), 1):
        cache = da.PagedCache(empty.keys.clone(), empty.values.clone())
        da.cache_append_hip(cache, key, value, s.table, s.lengths, s.offsets, max_chunk=hint)
        assert torch.equal(cache.keys, expected_k) and torch.equal(cache.values, expected_v)
    for b, n in enumerate(lengths):
        keys, values = s.cache.rows(s.table[b, :-(-n // page)], n)
        assert torch.equal(keys.double().cpu(), s.rows[b][0]) and torch.equal(values.double().cpu(), s.rows[b][1])


@pytest.mark.gpu
def test_cache_append_drops_what_has_no_place() -> None:
    s = Setup([100, 40], [100, 40], 1, 64, 64, 32)
    key, value = s.query, torch.ones(140, 64, dtype=torch.bfloat16, device="cuda")
    before = s.cache.keys.clone(), s.cache.values.clone()

    def unchanged() -> bool:
        return torch.equal(s.cache.keys.nan_to_num(9), before[0].nan_to_num(9)) and torch.equal(
            s.cache.values.nan_to_num(9), before[1].nan_to_num(9))

    for bad in (-1, 1 << 30, s.cache.keys.shape[0]):
        da.cache_append_hip(s.cache, key, value, torch.full_like(s.table, bad), s.lengths, s.offsets)
        assert unchanged()
    da.cache_append_hip(s.cache, key, value, s.table, torch.full_like(s.lengths, 1 << 30), s.offsets)
    assert unchanged()   # positions behind the table
    da.cache_append_hip(s.cache, key, value, s.table, torch.zeros_like(s.lengths), s.offsets)
    assert unchanged()   # positions in front of the sequence


@pytest.mark.gpu
def test_cache_append_strided_rows() -> None:
    s = Setup([70, 33], [70, 33], 2, 64, 128, 64)
    pairs = torch.stack((torch.zeros_like(s.query), s.query), 1)
    wide = torch.randn(103, 200, device="cuda").bfloat16()
    value = wide[:, 8:136]
    da.cache_append_hip(s.cache, pairs[:, 1], value, s.table, s.lengths, s.offsets)
    got_k, got_v = s.cache.rows(s.table[0, :2], 70)
    assert torch.equal(got_k, s.query[:70]) and torch.equal(got_v, value[:70])
    value = wide[:, 3:131]   # not aligned: copied by the call
    da.cache_append_hip(s.cache, s.query, value, s.table, s.lengths, s.offsets)
    assert torch.equal(s.cache.rows(s.table[1, :1], 33)[1], value[70:])


def plain_select(weights, lengths, keep, recent):
    kept = torch.full((len(lengths), keep), -1, dtype=torch.int32)
    counts = []
    for b, n in enumerate(lengths):
        n = max(0, min(n, weights.shape[1]))
        count = min(n, keep)
        r = min(recent, count)
        w = [(-math.inf if math.isnan(x) else x, not math.isnan(x)) for x in weights[b, :n - r].tolist()]
        order = sorted(range(n - r), key=lambda i: (not w[i][1], -w[i][0], i))[:count - r]
        chosen = sorted(order) + list(range(n - r, n))
        kept[b, :count] = torch.tensor(chosen, dtype=torch.int32)
        counts.append(count)
    return kept, torch.tensor(counts, dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 0), (1, 1), (7, 3), (64, 64), (100, 0), (513, 17), (5000, 100)])
def test_cache_select(keep, recent) -> None:
    device = _device()
    g = torch.Generator().manual_seed(keep)
    lengths = [0, 1, 6, 64, 65, 700, 1025, 4100, 5003]
    weights = torch.rand(len(lengths), 5003, generator=g) ** 6
    weights[:, 3::11] = 0.125                       # equal ones
    weights[2, :4] = torch.tensor([0.0, -0.0, 0.0, -1.0])
    weights[5] = 1.0                                # all equal
    weights[6] = -weights[6]
    weights[7, ::5] = math.nan
    weights[7, 1::5] = math.inf
    weights[7, 2::5] = -math.inf
    weights[8, 100:] = 1e-42                        # below the normal range
    expected = plain_select(weights, lengths, keep, recent)
    got = da.cache_select_hip(weights.to(device), torch.tensor(lengths, dtype=torch.int32, device=device), keep, recent)
    assert torch.equal(got[0].cpu(), expected[0]) and torch.equal(got[1].cpu(), expected[1])
    # A view of wider rows, lengths outside of [0, capacity].
    lengths = [5003 + 1, -1, 1 << 30, 3, 4, 5, 6, 7, 8]
    wide = torch.zeros(9, 6000, device=device)
    wide[:, 500:5503] = weights.to(device)
    expected = plain_select(weights, lengths, keep, recent)
    got = da.cache_select_hip(wide[:, 500:5503], torch.tensor(lengths, dtype=torch.int32, device=device), keep, recent)
    assert torch.equal(got[0].cpu(), expected[0]) and torch.equal(got[1].cpu(), expected[1])


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1024, 1025, 4096, 4097, 32768, 32769])
def test_cache_select_where_rows_stop_to_fit_registers(length) -> None:
    g = torch.Generator().manual_seed(length)
    weights = torch.rand(3, length, generator=g) ** 8
    weights[1] = (weights[1] * 20).floor()
    lengths = [length, length, length - 1]
    keep = length // 3
    expected = plain_select(weights, lengths, keep, 0)
    got = da.cache_select_hip(weights.to(_device()), torch.tensor(lengths, dtype=torch.int32, device="cuda"), keep, 0)
    assert torch.equal(got[0].cpu(), expected[0]) and torch.equal(got[1].cpu(), expected[1])


@pytest.mark.gpu
def test_cache_select_long() -> None:
    device = _device()
    weights = torch.rand(2, 140000, generator=torch.Generator().manual_seed(5)).to(device)
    weights[1] = (weights[1] * 50).floor()
    lengths = torch.tensor([140000, 131071], dtype=torch.int32, device=device)
    kept, counts = da.cache_select_hip(weights, lengths, 30000, 1000)
    for b, n in enumerate(lengths.tolist()):
        order = torch.sort(weights[b, :n - 1000], descending=True, stable=True).indices[:29000]
        assert torch.equal(kept[b, :29000].long(), order.sort().values)
        assert torch.equal(kept[b, 29000:].long(), torch.arange(n - 1000, n, device=device))
    assert counts.tolist() == [30000, 30000]


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("own_pool", [False, True])
@pytest.mark.parametrize("page,out_page,branches,routing_dim,value_dim", [(32, 32, 1, 64, 64), (64, 64, 2, 64, 576), (96, 96, 1, 256, 512),
                                                                         (32, 128, 1, 64, 64)])
def test_cache_compact(page, out_page, branches, routing_dim, value_dim, own_pool, types) -> None:
    if own_pool and page != out_page:
        page = out_page
    lengths = [5, 300, 64, 0, 129, 1000]
    keep = 131
    need = sum(-(-min(n, keep) // out_page) for n in lengths)
    s = Setup(lengths, [0] * 6, branches, routing_dim, value_dim, page, types, spare=need + 1)
    g = torch.Generator().manual_seed(0)
    weights = torch.rand(6, s.table.shape[1] * page, generator=g).cuda()
    kept, counts = da.cache_select_hip(weights, s.lengths, keep, 20)
    out_table = torch.full((6, -(-keep // out_page) + 1), -1, dtype=torch.int32)
    used = set(s.table.flatten().tolist())
    free = [p for p in range(s.cache.keys.shape[0]) if p not in used]
    for b, n in enumerate(lengths):
        for i in range(-(-min(n, keep) // out_page)):
            out_table[b, i] = free.pop()
    out_table = out_table.cuda()
    if own_pool:
        out = s.cache
    else:
        out = da.PagedCache(
            torch.full((s.cache.keys.shape[0], out_page, branches, routing_dim), 3.0, dtype=types[0], device="cuda"),
            torch.full((s.cache.keys.shape[0], out_page // 32, value_dim, 32), 3.0, dtype=types[1], device="cuda"))
    expected_k, expected_v = out.keys.clone(), out.values.clone()
    expected_w = torch.zeros(6, out_table.shape[1] * out_page)
    for b, n in enumerate(lengths):
        for i, t in enumerate(kept[b, :min(n, keep)].tolist()):
            at = int(out_table[b, i // out_page])
            expected_k[at, i % out_page] = s.rows[b][0][t].to(types[0]).cuda()
            expected_v[at, i % out_page // 32, :, i % 32] = s.rows[b][1][t].to(types[1]).cuda()
            expected_w[b, i] = weights[b, t]
    moved = da.cache_compact_hip(s.cache, s.table, kept, counts, out, out_table, weights=weights)
    assert torch.equal(moved.cpu(), expected_w)
    assert torch.equal(out.keys.nan_to_num(9), expected_k.nan_to_num(9))
    assert torch.equal(out.values.nan_to_num(9), expected_v.nan_to_num(9))


@pytest.mark.gpu
def test_cache_compact_places_that_are_not_there() -> None:
    s = Setup([100, 90], [0, 0], 1, 64, 64, 32)
    out = da.PagedCache(torch.zeros_like(s.cache.keys), torch.zeros_like(s.cache.values))
    kept = torch.tensor([[0, 5, 1 << 30, -7], [1, 2, 3, 4]], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0], [-1]], dtype=torch.int32, device="cuda")
    counts = torch.tensor([1 << 30, 4], dtype=torch.int32, device="cuda")
    assert da.cache_compact_hip(s.cache, s.table, kept, counts, out, table) is None
    assert torch.equal(out.keys[0, :2, 0].double().cpu(), s.rows[0][0][[0, 5], 0])
    assert torch.equal(out.values[0, 0, :, :2].T.double().cpu(), s.rows[0][1][[0, 5]])
    assert not out.keys[0, 2:].any() and not out.keys[1:].any() and not out.values[0, 0, :, 2:].any() and not out.values[1:].any()


# ---- log probabilities --------------------------------------------------------


def exact_scores(logits, tokens):
    x = logits.double()
    logs = torch.log_softmax(x, -1)
    p = logs.exp()
    chosen = logs.gather(-1, tokens.clamp(0, x.shape[-1] - 1).unsqueeze(-1)).squeeze(-1)
    entropy = -torch.where(p > 0, p * logs, torch.zeros_like(p)).sum(-1)
    return logs, chosen, torch.where(logs.isnan().any(-1), math.nan, entropy)


def score_tolerance(logits):
    """Absolute tolerances of log probabilities of size 1, per unit of size: the
    sum of exponentials is off by its additions (at most V / 256 in a row and a
    tree), by its exponentials' exponents (F32 times their size, which the
    weights keep below log V on average) and two steps each."""

    v = logits.shape[-1]
    return F32 * (v / 256 + 4 * math.log(v + 1) + 48)


def check_scores(got, logits, tokens, top):
    logs, chosen, entropy = exact_scores(logits, tokens)
    unit = score_tolerance(logits)
    finite = torch.nan_to_num(chosen, 0.0, 0.0, 0.0).abs()
    close(got.log_probs, chosen, unit + 4 * F32 * (finite + math.log(logits.shape[-1] + 1)))
    # H = log s - t / s; t is a sum like s, of terms whose size is below log V
    # plus what the reference may lie off the maximum.
    close(got.entropy, entropy, unit * (4 + 2 * math.log(logits.shape[-1] + 1)) + entropy.nan_to_num(0) * 4 * F32)
    if top:
        order = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[..., :top]
        assert torch.equal(got.top_tokens, order)
        expected = logs.gather(-1, order)
        close(got.top_log_probs, expected, unit + 4 * F32 * (expected.nan_to_num(0, 0, 0).abs() + math.log(logits.shape[-1] + 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 7, 0), (2, 64, 64), (9, 65, 5), (4, 511, 20), (7, 513, 1),
                                            (1, 2048, 5), (33, 2049, 3), (1, 50001, 20), (130, 5003, 33), (2, 131072, 64),
                                            (1100, 1000, 7)])
def test_token_log_probs(rows, vocab, top, dtype) -> None:
    device = _device()
    g = torch.Generator().manual_seed(rows + vocab)
    x = torch.randn(rows, vocab, generator=g) * 3
    x[torch.rand(rows, vocab, generator=g) < 0.01] += 8
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(device)
    logits = x.to(dtype).to(device)
    check_scores(da.token_log_probs_hip(logits, tokens, top=top), logits, tokens, top)
    # Rows at any address: a view of a wider matrix.
    wide = torch.full((rows, vocab + 13), math.nan, dtype=dtype, device=device)
    wide[:, 5:vocab + 5] = logits
    check_scores(da.token_log_probs_hip(wide[:, 5:vocab + 5], tokens, top=top), logits, tokens, top)
    plain = da.token_log_probs_hip(logits, tokens, entropy=False)
    assert plain.entropy is None and plain.top_tokens is None
    assert torch.equal(plain.log_probs, da.token_log_probs_hip(logits, tokens).log_probs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [70, 5000, 70001])
def test_token_log_probs_special_rows(vocab, dtype) -> None:
    device = _device()
    low, inf = torch.finfo(dtype).min, math.inf
    x = torch.randn(12, vocab, generator=torch.Generator().manual_seed(0))
    x[0] = 0.0                        # all equal
    x[1] = low                        # masked by the lowest value throughout
    x[2, 3:] = -inf                   # three tokens are left
    x[3] = -inf                       # none is
    x[4, 5] = math.nan
    x[5, 7] = inf
    x[6, : vocab // 2] = low
    x[7, -1] = torch.finfo(dtype).max
    x[8] = torch.linspace(-50, 50, vocab)
    x[9] = torch.linspace(50, -50, vocab)
    x[10, ::2], x[10, 1::2] = 0.0, -0.0
    x[11, -3:] = 30.0
    logits = x.to(dtype).to(device)
    tokens = torch.randint(0, 3, (12,), generator=torch.Generator().manual_seed(1)).to(device)
    got = da.token_log_probs_hip(logits, tokens, top=5)
    clean = [i for i in range(12) if i not in (4, 5)]
    part = type(got)(*(t[clean] for t in got))
    check_scores(part, logits[clean], tokens[clean], 5)
    assert got.log_probs[[4, 5]].isnan().all() and got.entropy[[4, 5]].isnan().all() and got.top_log_probs[[4, 5]].isnan().all()
    assert 5 not in got.top_tokens[4].tolist() and got.top_tokens[5, 0] == 7


@pytest.mark.gpu
def test_token_log_probs_ties_and_missing() -> None:
    device = _device()
    for vocab in (40, 3000, 40000):
        x = torch.zeros(3, vocab)
        x[1, 17::3] = 1.0
        x[2] = math.nan
        x[2, [30, 4, 9]] = torch.tensor([1.0, 1.0, 2.0])
        got = da.token_log_probs_hip(x.bfloat16().to(device), torch.zeros(3, dtype=torch.int64, device=device), top=6)
        assert got.top_tokens[0].tolist() == [0, 1, 2, 3, 4, 5]
        assert got.top_tokens[1].tolist() == [17, 20, 23, 26, 29, 32]
        assert got.top_tokens[2].tolist() == [9, 4, 30, -1, -1, -1]


@pytest.mark.gpu
def test_token_log_probs_tokens_outside() -> None:
    device = _device()
    logits = torch.randn(5, 300, device=device).requires_grad_()
    tokens = torch.tensor([3, -100, 300, -1, 299], device=device)
    got = da.token_log_probs_hip(logits, tokens)
    assert got.log_probs[1] == 0 and got.log_probs[[2, 3]].isnan().all() and not got.log_probs[[0, 4]].isnan().any()
    (grad,) = torch.autograd.grad(got.log_probs.sum(), logits)
    assert not grad[1].any() and grad[[2, 3]].isnan().all() and not grad[[0, 4]].isnan().any()
    got = da.token_log_probs_hip(logits.detach(), tokens, ignore_index=3)
    assert got.log_probs[0] == 0 and got.log_probs[1].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 9, 0), (4, 511, 5), (2, 2050, 0), (1, 50001, 8), (130, 5003, 3)])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_token_log_probs_gradient(rows, vocab, top, dtype, with_entropy) -> None:
    device = _device()
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(2, rows, vocab, generator=g) * 3).to(dtype).to(device).requires_grad_()
    tokens = torch.randint(0, vocab, (2, rows), generator=g).to(device)
    got = da.token_log_probs_hip(logits, tokens, top=top, entropy=with_entropy)
    g_lp, g_h = torch.randn(2, rows, generator=g).to(device), torch.randn(2, rows, generator=g).to(device)
    g_top = torch.randn(2, rows, top, generator=g).to(device)
    outputs, grads = [got.log_probs], [g_lp]
    if with_entropy:
        outputs, grads = outputs + [got.entropy], grads + [g_h]
    if top:
        outputs, grads = outputs + [got.top_log_probs], grads + [g_top]
    (grad,) = torch.autograd.grad(outputs, logits, grads)
    x = logits.detach().double().requires_grad_()
    logs = torch.log_softmax(x, -1)
    chosen = logs.gather(-1, tokens.unsqueeze(-1)).squeeze(-1)
    exact = [chosen]
    if with_entropy:
        exact.append(-(logs.exp() * logs).sum(-1))
    if top:
        exact.append(logs.gather(-1, got.top_tokens))
    (expected,) = torch.autograd.grad(exact, x, [t.double() for t in grads])
    # The formula's terms: -p (G + g_H (log p + H)) and what is added at a token.
    lp, p = logs.detach(), logs.detach().exp()
    h = -(p * lp).sum(-1, keepdim=True)
    big = g_lp.double().abs().unsqueeze(-1) + (g_top.double().abs().sum(-1, keepdim=True) if top else 0)
    eh = g_h.double().abs().unsqueeze(-1) if with_entropy else 0 * big
    unit = score_tolerance(logits)
    relative = 2 * unit + F32 * (4 * lp.abs() + 16 + 2 * top)
    tolerance = p * (big + eh * (h + lp.abs())) * relative + p * eh * (unit * (4 + 2 * math.log(vocab + 1)) + 8 * F32 * h)
    tolerance = tolerance + (half_step(dtype) + 4 * F32) * expected.abs() + 4 * F32 * big * (lp > -1e9)
    tolerance = tolerance + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    close(grad, expected, tolerance)


@pytest.mark.gpu
def test_token_log_probs_gradient_against_differences() -> None:
    device = _device()
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 40, generator=g).to(device)
    tokens = torch.tensor([3, 17], device=device)

    def loss(t):
        got = da.token_log_probs_hip(t, tokens, top=3)
        return got.log_probs.sum() + 0.5 * got.entropy.sum() + (got.top_log_probs * torch.tensor([1.0, -2.0, 0.5], device=device)).sum()

    leaf = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(loss(leaf), leaf)
    step = 2.0 ** -7
    for j in (0, 3, 17, 39):
        there, back = x.clone(), x.clone()
        there[:, j] += step
        back[:, j] -= step
        # Third derivatives of these sums stay below 8; the fp32 losses, of size
        # 30, are off by 100 F32 of it at most.
        difference = (loss(there) - loss(back)).item() / (2 * step)
        assert abs(difference - grad[:, j].sum().item()) <= 2 * 8 * step ** 2 + 100 * 30 * F32 / step


@pytest.mark.gpu
def test_token_log_probs_gradients_of_views() -> None:
    device = _device()
    base = torch.randn(6, 333, device=device)
    tokens = torch.arange(5, device=device)
    leaf = base.clone().requires_grad_()
    (expected,) = torch.autograd.grad(da.token_log_probs_hip(leaf[:5], tokens).log_probs.sum(), leaf)
    other = base.clone().requires_grad_()
    (got,) = torch.autograd.grad(da.token_log_probs_hip(other.T.contiguous().T[:5], tokens).log_probs.sum(), other)
    assert torch.equal(got, expected) and not got[5].any()
    # One row for several tokens: the gradients add up.
    row = torch.randn(1, 333, device=device).requires_grad_()
    (shared,) = torch.autograd.grad(da.token_log_probs_hip(row.expand(5, 333), tokens).log_probs.sum(), row)
    many = row.detach().repeat(5, 1).requires_grad_()
    (single,) = torch.autograd.grad(da.token_log_probs_hip(many, tokens).log_probs.sum(), many)
    close(shared[0], single.double().sum(0), 8 * F32 * single.double().abs().sum(0))


@pytest.mark.gpu
def test_offsets_beyond_32_bits() -> None:
    """Pages and logits behind 2^32 elements."""

    device = _device()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB")
    s = Setup([70, 33], [1, 1], 1, 64, 64, 32)
    pages = s.cache.keys.shape[0]
    far = torch.empty(((1 << 32) + 4096 * pages * 64), dtype=torch.float16, device=device)
    keys = far.as_strided(s.cache.keys.shape, ((1 << 32) // (pages - 1) // 8 * 8 + 8, 64, 64, 1))
    keys.copy_(s.cache.keys)
    expected, tolerance, _, _ = s.exact(scales_of(1))
    got = da.paged_attention_hip(s.query, da.PagedCache(keys, s.cache.values), s.table, s.lengths, s.offsets, scales_of(1).to(device))
    close(got.cpu(), expected, tolerance)
    del far, keys
    rows = torch.zeros((1 << 32) // 65536 + 3, 65536, dtype=torch.bfloat16, device=device)
    rows[-1, 7] = 20.0
    tokens = torch.full((rows.shape[0],), 7, dtype=torch.int64, device=device)
    got = da.token_log_probs_hip(rows, tokens, top=1)
    assert got.top_tokens[-1, 0] == 7 and got.top_tokens[-2, 0] == 0 and got.log_probs[-1] > -0.01 > got.log_probs[-2]


@pytest.mark.gpu
def test_serving_step_as_a_graph() -> None:
    """Append, attention with weights, selection and move, captured and replayed
    on changing inputs, against eager calls of the same inputs."""

    s = Setup([200, 90, 333], [5, 1, 40], 2, 64, 128, 32, spare=20)
    value = torch.randn(46, 128, device="cuda").bfloat16()
    key = torch.randn_like(s.query)
    scales = scales_of(2).cuda()
    used = set(s.table.flatten().tolist())
    free = [p for p in range(s.cache.keys.shape[0]) if p not in used]
    out_table = torch.tensor(free[:12], dtype=torch.int32, device="cuda").view(3, 4)
    before = torch.rand(3, s.table.shape[1] * 32, device="cuda")

    def step(cache):
        da.cache_append_hip(cache, key, value, s.table, s.lengths, s.offsets, max_chunk=40)
        out, weights = da.paged_attention_weights_hip(*((s.query, cache) + s.where()[2:]), scales, weights=before, max_chunk=40)
        kept, counts = da.cache_select_hip(weights, s.lengths, 100, 10)
        moved = da.cache_compact_hip(cache, s.table, kept, counts, cache, out_table, weights=weights)
        return out, weights, kept, counts, moved, cache.keys, cache.values

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s.cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(s.cache)
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        s.query.copy_(torch.nn.functional.normalize(torch.randn(s.query.shape, generator=g), dim=-1))
        key.copy_(torch.nn.functional.normalize(torch.randn(key.shape, generator=g), dim=-1))
        s.lengths.copy_(torch.tensor([200 - i, 90 - i, 333 - 7 * i], dtype=torch.int32))
        cache = da.PagedCache(s.cache.keys.clone(), s.cache.values.clone())
        eager = step(cache)
        torch.cuda.synchronize()
        graph.replay()
        for got, expected in zip(captured, eager):
            assert torch.equal(got.nan_to_num(9.0), expected.nan_to_num(9.0))


@pytest.mark.gpu
def test_training_step_as_a_graph() -> None:
    device = _device()
    logits = torch.randn(64, 5000, device=device).bfloat16()
    tokens = torch.randint(0, 5000, (64,), device=device)
    leaf = logits.clone().requires_grad_()
    eager_graph = da.token_log_probs_hip(leaf, tokens)   # another leaf's graph stays alive
    static = logits.clone().requires_grad_()

    def step():
        got = da.token_log_probs_hip(static, tokens)
        return torch.autograd.grad(got.log_probs.mean() + got.entropy.mean(), static)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        with torch.no_grad():
            static.copy_(torch.randn(64, 5000, device=device).bfloat16())
        expected = step()
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(captured, expected)
    torch.autograd.grad(eager_graph.log_probs.sum(), leaf)


@pytest.mark.gpu
def test_two_streams_at_once() -> None:
    a = Setup([2000, 900], [1, 1], 1, 256, 512, 64, seed=1)
    b = Setup([700, 1500], [60, 130], 1, 256, 512, 64, seed=2)
    scales = scales_of(1).cuda()
    expected = [da.paged_attention_hip(*s.where(), scales) for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(da.paged_attention_hip(*s.where(), scales))
    torch.cuda.synchronize()
    assert all(torch.equal(x, expected[i]) for i in range(2) for x in got[i])


# ---- refusals (on the CPU) ------------------------------------------------------

HEADER = Path(__file__).resolve().parents[1] / "include" / "double_attention_serving.h"


def test_header_declares_what_is_bound() -> None:
    text = HEADER.read_text()
    names = set(re.findall(r"\b(da_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(_lib.SERVING_SIGNATURES)
    assert f"#define DA_MAX_TOP {serving_ops.MAX_TOP}" in text
    for limit in (serving_ops.MAX_PAGE_SIZE, serving_ops.MAX_KEY_WIDTH, serving_ops.MAX_VALUE_DIM):
        assert f"up to {limit}" in text


PTR = 1 << 20


def _cache(**changes):
    values = dict(keys=PTR, key_page_stride=64 * 64, values=2 * PTR, value_page_stride=64 * 128, pages=4, page_size=64, key_width=64,
                  value_dim=128, page_table=3 * PTR, ld_table=4, table_pages=4)
    values.update(changes)
    return _lib.PagedCacheArgs(*values.values())


BAD_CACHES = [
    (dict(page_size=48), -2, "page_size 48"), (dict(page_size=8192), -2, "page_size 8192"), (dict(key_width=96), -2, "key_width 96"),
    (dict(key_width=2048), -2, "key_width 2048"), (dict(value_dim=96), -2, "value_dim 96"), (dict(value_dim=5120), -2, "value_dim"),
    (dict(pages=0), -1, "no pages"), (dict(table_pages=5), -1, "fewer entries"), (dict(keys=0), -1, "null"), (dict(values=0), -1, "null"),
    (dict(page_table=0), -1, "null"), (dict(keys=PTR + 8), -3, "aligned"), (dict(key_page_stride=64 * 64 + 4), -3, "multiples of 8"),
    (dict(key_page_stride=64 * 32), -1, "at least a page"), (dict(value_page_stride=64 * 64), -1, "at least a page"),
    (dict(table_pages=1 << 30, ld_table=1 << 30), -1, "2\\^27"),
]


@pytest.mark.parametrize("changes,code,pattern", BAD_CACHES)
def test_c_entries_refuse_bad_caches(changes, code, pattern) -> None:
    h = _lib.get()
    cache = _cache(**changes)
    assert h.da_cache_append(cache, 4 * PTR, 64, 5 * PTR, 128, 3, 6 * PTR, 7 * PTR, 2, 0, None) == code
    assert re.search(pattern, h.da_last_error().decode())
    args = _attention()
    args.cache = cache
    assert h.da_paged_attention(args, None) == code and re.search(pattern, h.da_last_error().decode())
    assert h.da_paged_attention_workspace_bytes(args) == 0 or "null" in pattern or code == -3 or "at least" in pattern
    other = _cache(keys=10 * PTR, values=11 * PTR)
    for pair in ((cache, other), (other, cache)):
        assert h.da_cache_compact(*pair, 2, 4 * PTR, 8, 8, 5 * PTR, None, 0, None, 0, None) == code


def _attention(**changes):
    values = dict(cache=_cache(), query=4 * PTR, ldq=64, rows=3, lengths=6 * PTR, offsets=7 * PTR, sequences=2, scales=8 * PTR,
                  scales_dtype=0, scale_mult=1.0, maps=1, score_dim=64, map_repeat=1, causal=1, mix=0, qk_dtype=_lib.DA_F16,
                  v_dtype=_lib.DA_BF16, out=9 * PTR, weights_in=0, weights_out=0, ld_weights=256, max_chunk=0, max_length=0,
                  workspace=12 * PTR, workspace_bytes=1 << 19)
    values.update(changes)
    return _lib.PagedAttentionArgs(*values.values())


@pytest.mark.parametrize("changes,code,pattern", [
    (dict(qk_dtype=_lib.DA_BF16, v_dtype=_lib.DA_F16), -2, "qk_dtype"), (dict(qk_dtype=_lib.DA_F32), -2, "qk_dtype"),
    (dict(maps=0), -2, "maps"), (dict(maps=65), -2, "maps"), (dict(score_dim=96), -2, "score_dim"), (dict(score_dim=576), -2, "score_dim"),
    (dict(maps=2), -1, "do not fit"), (dict(map_repeat=2), -1, "do not fit"), (dict(scales_dtype=9), -1, "scales"),
    (dict(scale_mult=float("nan")), -1, "scales"), (dict(rows=-1), -2, "rows"), (dict(rows=1 << 23), -2, "rows"),
    (dict(lengths=0), -1, "lengths"), (dict(offsets=7 * PTR + 2), -1, "offsets"), (dict(query=0), -1, "query"),
    (dict(query=4 * PTR + 8), -3, "query"), (dict(ldq=60), -3, "query"), (dict(ldq=56), -3, "query"), (dict(scales=0), -1, "scales"),
    (dict(out=0), -3, "out"), (dict(out=9 * PTR + 8), -3, "out"), (dict(weights_out=13 * PTR, ld_weights=255), -1, "weights"),
    (dict(weights_out=13 * PTR + 1), -1, "weights"), (dict(workspace=0, weights_out=13 * PTR), -5, "workspace"),
    (dict(workspace_bytes=16, weights_out=13 * PTR), -5, "workspace"), (dict(workspace=12 * PTR + 8, weights_out=13 * PTR), -3, "workspace"),
    (dict(out=PTR), -1, "overlaps"), (dict(out=2 * PTR + 32), -1, "overlaps"), (dict(out=4 * PTR), -1, "overlaps"),
    (dict(weights_out=6 * PTR), -1, "overlaps"), (dict(weights_out=13 * PTR, weights_in=13 * PTR + 64), -1, "overlaps"),
    (dict(sequences=70000), -2, "sequences"), (dict(sequences=-1), -2, "sequences"), (dict(sequences=0), -1, "without sequences"),
])
def test_c_attention_refuses(changes, code, pattern) -> None:
    h = _lib.get()
    assert h.da_paged_attention(_attention(**changes), None) == code
    assert re.search(pattern, h.da_last_error().decode())


def test_c_cache_moves_refuse() -> None:
    h = _lib.get()

    def append(**changes):
        a = dict(cache=_cache(), key=4 * PTR, ldk=64, value=5 * PTR, ldv=128, rows=3, lengths=6 * PTR, offsets=7 * PTR, sequences=2,
                 max_chunk=0, stream=None)
        a.update(changes)
        return h.da_cache_append(*a.values())

    for changes, code in ((dict(cache=None), -1), (dict(key=0), -1), (dict(key=4 * PTR + 2), -3), (dict(ldk=63), -3), (dict(ldk=56), -3),
                          (dict(value=0), -1), (dict(ldv=120), -3), (dict(rows=-1), -2), (dict(lengths=0), -1), (dict(offsets=0), -1),
                          (dict(key=PTR), -1), (dict(value=2 * PTR), -1), (dict(lengths=PTR + 64), -1), (dict(rows=0), 0),
                          (dict(sequences=0), 0)):
        assert append(**changes) == code, changes

    def select(**changes):
        a = dict(weights=PTR, ld=100, capacity=100, lengths=2 * PTR, sequences=2, keep=10, recent=2, kept=3 * PTR, counts=4 * PTR, stream=None)
        a.update(changes)
        return h.da_cache_select(*a.values())

    for changes, code in ((dict(weights=0), -1), (dict(ld=99), -1), (dict(capacity=-1), -2), (dict(capacity=1 << 40), -2),
                          (dict(lengths=0), -1), (dict(keep=-1), -1), (dict(recent=11), -1), (dict(recent=-1), -1), (dict(kept=0), -1),
                          (dict(counts=0), -1), (dict(counts=4 * PTR + 2), -3), (dict(kept=PTR), -1), (dict(counts=3 * PTR + 16), -1),
                          (dict(sequences=1 << 20), -2), (dict(sequences=0), 0)):
        assert select(**changes) == code, changes

    def compact(**changes):
        a = dict(source=_cache(), to=_cache(keys=10 * PTR, values=11 * PTR), sequences=2, kept=4 * PTR, ld_kept=8, keep=8, counts=5 * PTR,
                 win=6 * PTR, ld_in=256, wout=7 * PTR, ld_out=256, stream=None)
        a.update(changes)
        return h.da_cache_compact(*a.values())

    for changes, code in ((dict(source=None), -1), (dict(to=None), -1), (dict(to=_cache(keys=10 * PTR, key_width=128, key_page_stride=64 * 128)), -1),
                          (dict(kept=0), -1), (dict(ld_kept=7), -1), (dict(counts=0), -1), (dict(win=0), -1), (dict(ld_in=255), -1),
                          (dict(ld_out=255), -1), (dict(wout=6 * PTR + 64), -1), (dict(wout=10 * PTR), -1),
                          (dict(to=_cache(keys=PTR + 1024, values=11 * PTR)), -1), (dict(to=_cache(keys=2 * PTR, values=11 * PTR)), -1),
                          (dict(to=_cache(keys=10 * PTR, page_size=32, table_pages=4)), -1), (dict(sequences=0), 0)):
        assert compact(**changes) == code, changes


def test_c_token_log_probs_refuses() -> None:
    h = _lib.get()

    def forward(**changes):
        a = dict(logits=PTR, rows=4, vocab=1000, ldx=1000, dtype=_lib.DA_BF16, tokens=2 * PTR, ignore=-100, log_probs=3 * PTR, entropy=0,
                 lse=0, top=5, top_lp=4 * PTR, top_tokens=5 * PTR, workspace=6 * PTR, nbytes=1 << 19, stream=None)
        a.update(changes)
        return h.da_token_log_probs(*a.values())

    for changes, code in ((dict(logits=0), -3), (dict(logits=PTR + 1), -3), (dict(rows=-1), -2), (dict(vocab=0), -2), (dict(vocab=1 << 25), -2),
                          (dict(ldx=999), -1), (dict(dtype=7), -1), (dict(tokens=0), -1), (dict(log_probs=0), -1), (dict(top=65), -2),
                          (dict(top=-1), -2), (dict(vocab=4, ldx=4), -2), (dict(top_lp=0), -1), (dict(top_tokens=0), -1),
                          (dict(tokens=2 * PTR + 4), -3), (dict(log_probs=PTR), -1), (dict(entropy=3 * PTR), -1),
                          (dict(rows=1, vocab=1 << 20, ldx=1 << 20, logits=64 * PTR, workspace=0), -5), (dict(rows=0), 0)):
        assert forward(**changes) == code, changes

    def backward(**changes):
        a = dict(logits=PTR, rows=4, vocab=1000, ldx=1000, dtype=_lib.DA_BF16, tokens=2 * PTR, ignore=-100, lse=3 * PTR, entropy=4 * PTR, top=5,
                 top_tokens=5 * PTR, g_lp=6 * PTR, g_h=7 * PTR, g_top=8 * PTR, grad=9 * PTR, ldg=1000, stream=None)
        a.update(changes)
        return h.da_token_log_probs_backward(*a.values())

    for changes, code in ((dict(lse=0), -1), (dict(entropy=0), -1), (dict(top_tokens=0), -1), (dict(top=0), -1), (dict(grad=0), -3),
                          (dict(ldg=999), -1), (dict(grad=PTR), -1), (dict(grad=6 * PTR), -1), (dict(tokens=0), -1), (dict(rows=0), 0)):
        assert backward(**changes) == code, changes


def test_python_refuses_on_the_cpu() -> None:
    cache = da.paged_cache(4, 64, 2, 64, 128)
    assert cache.page_size == 64 and cache.keys.shape == (4, 64, 2, 64) and cache.values.shape == (4, 2, 128, 32)
    table, lengths = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    offsets = torch.tensor([0, 1, 2], dtype=torch.int32)
    q, v, scales = torch.zeros(2, 2, 64).half(), torch.zeros(2, 128).bfloat16(), torch.ones(2)
    for call in (
        lambda: da.cache_append_hip(cache, q, v, table, lengths, offsets),
        lambda: da.paged_attention_hip(q, cache, table, lengths, offsets, scales),
        lambda: da.paged_attention_weights_hip(q, cache, table, lengths, offsets, scales),
        lambda: da.cache_select_hip(torch.zeros(2, 128), lengths, 4),
        lambda: da.cache_compact_hip(cache, table, table, lengths, cache, table),
        lambda: da.token_log_probs_hip(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64)),
    ):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    for bad in (dict(pages=0), dict(page_size=33), dict(page_size=0), dict(branches=40), dict(routing_dim=10), dict(value_dim=8)):
        sizes = dict(pages=4, page_size=64, branches=2, routing_dim=64, value_dim=128)
        sizes.update(bad)
        with pytest.raises((ValueError, NotImplementedError)):
            da.paged_cache(**sizes)
    with pytest.raises(ValueError):
        da.paged_cache(4, 64, 2, 64, 128, key_dtype=torch.bfloat16, dtype=torch.float16)
    logits, tokens = torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64)
    for bad in ((logits.double(), tokens), (logits, tokens.int()), (logits, tokens[:1]), (logits[:, :0], tokens), (logits[0, 0], tokens[0])):
        with pytest.raises(ValueError):
            da.token_log_probs_hip(*bad)
    for top in (-1, 10, 65):
        with pytest.raises(NotImplementedError):
            da.token_log_probs_hip(logits, tokens, top=top)


@pytest.mark.gpu
def test_python_refuses() -> None:
    s = Setup([70, 33], [2, 1], 2, 64, 128, 32)
    scales = scales_of(2).cuda()
    query, cache, table, lengths, offsets = s.where()

    def refused(match, *where, error=ValueError, **kwargs):
        with pytest.raises(error, match=match):
            da.paged_attention_weights_hip(*where, **kwargs)

    refused("query is", query.bfloat16(), cache, table, lengths, offsets, scales)
    refused("query is", query[:, :1], cache, table, lengths, offsets, scales)
    refused("page_table", query, cache, table.long(), lengths, offsets, scales)
    refused("page_table on", query, cache, table.cpu(), lengths, offsets, scales)
    refused("lengths", query, cache, table, lengths[:1], offsets, scales)
    refused("lengths", query, cache, table, lengths.long(), offsets, scales)
    refused("offsets", query, cache, table, lengths, offsets[:2], scales)
    refused("scales", query, cache, table, lengths, offsets, scales.long())
    refused("scales", query, cache, table, lengths, offsets, scales[0])
    refused("maps of", query, cache, table, lengths, offsets, scales_of(3).cuda(), error=NotImplementedError)
    refused("mix is", query, cache, table, lengths, offsets, scales, mix=scales[:1])
    refused("weights is", query, cache, table, lengths, offsets, scales, weights=torch.zeros(2, 5, device="cuda"))
    refused("out is", query, cache, table, lengths, offsets, scales, out=torch.zeros(2, 5, device="cuda"))
    refused("max_chunk", query, cache, table, lengths, offsets, scales, max_chunk=0)
    refused("autograd", query.clone().requires_grad_(), cache, table, lengths, offsets, scales)
    refused("autograd", query, cache, table, lengths, offsets, scales.clone().requires_grad_())
    refused("a cache is", query, da.PagedCache(cache.keys, cache.values[..., :16]), table, lengths, offsets, scales)
    refused("contiguous", query, da.PagedCache(cache.keys.transpose(1, 2).contiguous().transpose(1, 2), cache.values), table, lengths, offsets, scales)
    refused("keys of", query, da.PagedCache(cache.keys.float(), cache.values), table, lengths, offsets, scales)
    with torch.autograd.forward_ad.dual_level():
        refused("forward-mode", torch.autograd.forward_ad.make_dual(query, query), cache, table, lengths, offsets, scales)
        with pytest.raises(ValueError, match="forward-mode"):
            x = torch.zeros(2, 9, device="cuda")
            da.token_log_probs_hip(torch.autograd.forward_ad.make_dual(x, x), torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="key is"):
        da.cache_append_hip(cache, query.float(), torch.zeros(3, 128, device="cuda").bfloat16(), table, lengths, offsets)
    with pytest.raises(ValueError, match="value is"):
        da.cache_append_hip(cache, query, torch.zeros(2, 128, device="cuda").bfloat16(), table, lengths, offsets)
    with pytest.raises(ValueError, match="recent"):
        da.cache_select_hip(torch.zeros(2, 128, device="cuda"), lengths, 4, 5)
    kept, counts = da.cache_select_hip(torch.zeros(2, 96, device="cuda"), lengths, 4)
    other = da.paged_cache(4, 32, 1, 64, 128, device="cuda")
    with pytest.raises(ValueError, match="widths"):
        da.cache_compact_hip(cache, table, kept, counts, other, table)
    with pytest.raises(ValueError, match="weights are"):
        da.cache_compact_hip(cache, table, kept, counts, cache, table, weights=torch.zeros(2, 5, device="cuda"))
    with pytest.raises(ValueError, match="overlaps"):
        da.cache_append_hip(cache, cache.keys.view(-1, 2, 64)[:3], torch.zeros(3, 128, device="cuda").bfloat16(), table, lengths, offsets)
