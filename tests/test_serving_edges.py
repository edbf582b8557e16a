"""Serving operators at values and sizes off the usual range, against 64-bit forms."""

from __future__ import annotations

import math

import pytest
import torch

import double_attention as da
from test_serving_ops import F32, TYPES, Setup, close, half_step, scales_of, score_tolerance

# ---- the gradient of log probabilities ---------------------------------------


def check_gradient(logits, tokens, top) -> None:
    """Against -p (G + g_H (log p + H)) and what is added at the named tokens, in 64 bits."""

    g = torch.Generator().manual_seed(logits.shape[-1])
    rows, vocab = logits.shape
    g_lp, g_h = (torch.randn(rows, generator=g).to(logits.device) for _ in range(2))
    g_top = torch.randn(rows, top, generator=g).to(logits.device)
    leaf = logits.clone().requires_grad_()
    got = da.token_log_probs_hip(leaf, tokens, top=top)
    outputs, grads = [got.log_probs, got.entropy], [g_lp, g_h]
    if top:
        outputs, grads = outputs + [got.top_log_probs], grads + [g_top]
    (grad,) = torch.autograd.grad(outputs, leaf, grads)
    lp = torch.log_softmax(logits.double(), -1)
    p = lp.exp()
    lp = torch.where(p == 0, 0.0, lp)   # no weight (a NaN stays)
    h = -(p * lp).sum(-1, keepdim=True)
    named = torch.zeros_like(p).scatter_add_(1, tokens[:, None], g_lp.double()[:, None])
    if top:
        named.scatter_add_(1, got.top_tokens, g_top.double())
    whole = g_lp.double()[:, None] + g_top.double().sum(-1, keepdim=True)
    eh = g_h.double()[:, None]
    expected = named - p * (whole + eh * (lp + h))
    # The terms of test_serving_ops.test_token_log_probs_gradient.
    big = g_lp.double().abs()[:, None] + g_top.double().abs().sum(-1, keepdim=True)
    unit = score_tolerance(logits)
    relative = 2 * unit + F32 * (4 * lp.abs() + 16 + 2 * top)
    tolerance = p * (big + eh.abs() * (h + lp.abs())) * relative
    tolerance = tolerance + p * eh.abs() * (unit * (4 + 2 * math.log(vocab + 1)) + 8 * F32 * h)
    tolerance = tolerance + (half_step(logits.dtype) + 4 * F32) * expected.abs() + 4 * F32 * big
    tolerance = tolerance + torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps
    close(grad, expected, tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1e4, -1e5, 1e5, 1e6])
@pytest.mark.parametrize("rows,vocab,top", [(3, 32000, 5), (260, 1000, 0)])
def test_gradient_of_logits_far_from_zero(rows, vocab, top, offset) -> None:
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 3 + offset).cuda()
    check_gradient(logits, torch.randint(0, vocab, (rows,), generator=g).cuda(), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [70, 5000, 70001])
def test_gradient_of_special_rows(vocab, dtype) -> None:
    low = torch.finfo(dtype).min
    x = torch.randn(8, vocab, generator=torch.Generator().manual_seed(0))
    x[0] = 0.0                                # all equal
    x[1] = low                                # masked by the lowest value throughout
    x[2, 3:] = -math.inf                      # three tokens are left
    x[3] = -math.inf                          # none is
    x[4, : vocab // 2] = low
    x[5, -1] = torch.finfo(dtype).max
    x[6] = torch.linspace(-50, 50, vocab)
    x[7] = low / 2
    tokens = torch.randint(0, 3, (8,), generator=torch.Generator().manual_seed(1)).cuda()
    check_gradient(x.to(dtype).cuda(), tokens, 2)


# ---- infinities and NaN in the cache -----------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lengths,chunks,layout,value_dim,mixed", [
    pytest.param([90, 40], [40, 3], (1, 1, 64), 64, False, id="few"),
    pytest.param([700, 40], [20, 1], (2, 2, 128), 320, True, id="few-in-parts"),
    pytest.param([700, 40], [20, 1], (1, 2, 64), 1088, False, id="few-in-slices"),
    pytest.param([640, 40], [600, 1], (1, 1, 64), 192, False, id="chunk"),
    pytest.param([2000, 40], [530, 1], (2, 2, 192), 576, True, id="chunk-in-parts"),
    pytest.param([700, 40], [640, 40], (1, 1, 512), 64, False, id="chunk-of-wide-keys"),
])
def test_a_value_reaches_the_rows_that_see_it(lengths, chunks, layout, value_dim, mixed, types, bad) -> None:
    branches, maps, routing_dim = layout
    s = Setup(lengths, chunks, branches, routing_dim, value_dim, 32, types)
    scales = scales_of(maps)
    mix = torch.softmax(torch.arange(maps, dtype=torch.float32), 0) if mixed else None
    expected, tolerance, weights, w_tolerance = s.exact(scales, True, mix)
    length, new = lengths[0], chunks[0]
    # New tokens at and off the tiles' borders, an old one, and the last one.
    for position in sorted({length - new - 1, length - new + 1, (length - new) // 32 * 32 + 32, length - 9, length - 1} & set(range(length))):
        feature = (position * 7) % value_dim
        at = (int(s.table[0, position // 32]), 0, feature, position % 32)
        held = s.cache.values[at].clone()
        s.cache.values[at] = bad
        got, gathered = da.paged_attention_weights_hip(*s.where(), scales.cuda(), mix=None if mix is None else mix.cuda(),
                                                       max_chunk=max(chunks))
        s.cache.values[at] = held
        got = got.cpu()
        seen = torch.zeros(s.total, dtype=torch.bool)
        seen[max(0, position - (length - new)):new] = True
        assert not got[seen][..., feature].isfinite().any()
        there = torch.zeros_like(got, dtype=torch.bool)
        there[seen, ..., feature] = True
        close(torch.where(there, 0, got), torch.where(there, 0.0, expected), tolerance)
        close(gathered.cpu(), weights, w_tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lengths,chunks,layout", [
    pytest.param([90, 40], [40, 3], (2, 2, 64), id="few"),
    pytest.param([90, 40], [9, 3], (4, 4, 128), id="few-of-512"),
    pytest.param([300, 40], [9, 3], (4, 2, 192), id="few-of-768"),
    pytest.param([90, 40], [3, 1], (2, 4, 64), id="few-shared"),
    pytest.param([640, 40], [600, 1], (2, 2, 64), id="chunk"),
])
def test_a_key_reaches_the_rows_and_maps_that_see_it(lengths, chunks, layout, types) -> None:
    branches, maps, routing_dim = layout
    s = Setup(lengths, chunks, branches, routing_dim, 128, 32, types)
    scales = scales_of(maps)
    expected, tolerance, weights, w_tolerance = s.exact(scales)
    length, new = lengths[0], chunks[0]
    for bad in (math.nan, math.inf, -math.inf):
        for position in (length - new + 1, length - 1):
            branch = branches - 1
            at = (int(s.table[0, position // 32]), position % 32, branch, 5)
            held = s.cache.keys[at].clone()
            s.cache.keys[at] = bad
            got, gathered = da.paged_attention_weights_hip(*s.where(), scales.cuda(), max_chunk=max(chunks))
            s.cache.keys[at] = held
            got = got.cpu()
            seen = torch.zeros(s.total, dtype=torch.bool)
            seen[position - (length - new):new] = True
            touched = torch.arange(maps) * branches // maps
            touched = (touched <= branch) & (branch < touched + max(1, branches // maps))
            there = (seen[:, None] & touched)[..., None].expand_as(got)
            if math.isnan(bad):
                assert got[there].isnan().all()
            close(torch.where(there, 0, got), torch.where(there, 0.0, expected), tolerance)
            close(gathered[1:].cpu(), weights[1:], w_tolerance[1:])


# ---- probabilities at the lower end of fp16 ----------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("below", [23.4, 24.6, 25.1, 27.0])
@pytest.mark.parametrize("chunk,length", [(1, 131072), (600, 16384)])
def test_a_long_flat_tail_beside_one_token_in_fp16(chunk, length, below) -> None:
    """One token of probability near one and value zero, and all others 2^-below
    of it with value one: what the tail has together is not lost or rounded up."""

    device = torch.device("cuda")
    # A scale of below / log2(e): the first key is the query, the others are half of
    # it beside a query of length two.
    keys = torch.zeros(length // 64, 64, 1, 64, dtype=torch.float16, device=device)
    keys[..., 0] = 0.5
    keys[0, 0, 0, 0] = 1.0
    values = torch.ones(length // 64, 2, 64, 32, dtype=torch.float16, device=device)
    values[0, 0, :, 0] = 0.0
    query = torch.zeros(chunk, 1, 64, dtype=torch.float16, device=device)
    query[..., 0] = 2.0
    table = torch.arange(length // 64, dtype=torch.int32, device=device)[None]
    lengths = torch.tensor([length], dtype=torch.int32, device=device)
    offsets = torch.tensor([0, chunk], dtype=torch.int32, device=device)
    scale = torch.tensor([below * math.log(2.0)])
    # One part for all tokens (a part has a reference of its own).
    got = da.paged_attention_hip(query, da.PagedCache(keys, values), table, lengths, offsets, scale.to(device), max_chunk=chunk, max_length=1)
    each = math.exp(-float(scale.double()))
    tail = each * (torch.arange(length - chunk, length, dtype=torch.float64))
    expected = (tail / (1 + tail))[:, None, None].expand(chunk, 1, 64)
    # A probability is off by half a step of fp16, or by 2^-25 where it is below
    # the normal range; the reference lies more than 6 below the largest score, so
    # that its probability is more than 2^6 beside that.  Scores of up to 54 (log2)
    # are off by three roundings each.
    tolerance = expected * (2 * half_step(torch.float16) + 2.0 ** -17) + length * 2.0 ** -25 / 2 ** 6 + 2.0 ** -25
    close(got.cpu(), expected, tolerance)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("chunk", [1, 40, 600])
@pytest.mark.parametrize("step", [0.3, 7.9, 8.1, 14.9, 15.1, 40.0])
def test_scores_that_rise_from_tile_to_tile(step, chunk, types) -> None:
    """Scores that stay just below and go just above what moves a reference, up and
    down along the sequence: nothing overflows the probabilities' type."""

    device, length, page = torch.device("cuda"), 1000, 32
    g = torch.Generator().manual_seed(0)
    tile = torch.arange(length) // 32
    level = torch.where(tile < 20, tile, 40 - tile) / 32 + torch.rand(length, generator=g) / 512
    keys = torch.zeros(page, page, 1, 64, dtype=types[0])
    keys.view(-1, 64)[:length, 0] = level.to(types[0])
    values = torch.randn(page * page, 64, generator=g).to(types[1])
    query = torch.zeros(chunk, 1, 64, dtype=types[0], device=device)
    query[..., 0] = 2.0
    scale = torch.tensor([step * 16 * math.log(2.0)])   # two times 1/32 of it: `step` in log2
    cache = da.PagedCache(keys.to(device), values.view(page, 1, 32, 64).transpose(2, 3).contiguous().to(device))
    table = torch.arange(page, dtype=torch.int32, device=device)[None]
    lengths = torch.tensor([length], dtype=torch.int32, device=device)
    offsets = torch.tensor([0, chunk], dtype=torch.int32, device=device)
    scores = (2 * keys.view(-1, 64)[:length, 0].double() * scale.double()).expand(chunk, length)
    seen = torch.arange(length)[None] <= torch.arange(length - chunk, length)[:, None]
    p = torch.softmax(scores.masked_fill(~seen, -math.inf), -1)
    v = values[:length].double()
    half = half_step(types[1])
    # A score is one exact product, times a scale of three roundings, and the
    # difference to the reference; scores reach 20 steps.
    delta = 8 * F32 * (20 * step + 1)
    tolerance = (half + 2 * delta + 16 * F32) * (p @ v.abs()) + half * (p @ v).abs() + 2.0 ** -25
    if types[1] is torch.float16:
        tolerance = tolerance + length * 2.0 ** -25 / 2 ** 6 * 5
    for max_length in (None, 1):
        got = da.paged_attention_hip(query, cache, table, lengths, offsets, scale.to(device), max_chunk=chunk, max_length=max_length)
        close(got[:, 0].cpu(), p @ v, tolerance)


# ---- launches --------------------------------------------------------------------


@pytest.mark.gpu
def test_many_sequences_of_many_maps_and_wide_values() -> None:
    """One token of each of 16384 sequences, 64 maps, 4096 value features, without a
    word on the chunks: workgroups for a chunk of each would be 2^32 threads."""

    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GiB")
    sequences, maps, page = 16384, 64, 32
    g = torch.Generator().manual_seed(0)
    cache = da.PagedCache(torch.randn(2, page, 1, 64, generator=g).half().cuda() / 8, torch.randn(2, 1, 4096, 32, generator=g).bfloat16().cuda())
    table = (torch.arange(sequences, dtype=torch.int32) % 2)[:, None].cuda()
    lengths = torch.full((sequences,), page, dtype=torch.int32, device="cuda")
    offsets = torch.arange(sequences + 1, dtype=torch.int32, device="cuda")
    query = torch.randn(2, 1, 64, generator=g).half().cuda().repeat(sequences // 2, 1, 1)
    scales = scales_of(maps, 1.0).cuda()
    got = da.paged_attention_hip(query, cache, table, lengths, offsets, scales)
    two = da.paged_attention_hip(query[:2], cache, table[:2], lengths[:2], offsets[:3], scales)
    assert bool(two.any()) and torch.equal(got.view(sequences // 2, 2, maps, 4096), two.expand(sequences // 2, 2, maps, 4096))


# ---- views ----------------------------------------------------------------------


@pytest.mark.gpu
def test_pages_of_one_branch_or_tile_with_any_stride_there() -> None:
    """The stride of a dimension of size one says nothing about the memory."""

    s = Setup([70, 33], [3, 1], 1, 64, 128, 32)
    pages = s.cache.keys.shape[0]
    keys = torch.full((pages, 3, 1, 32, 64), math.nan, dtype=torch.float16, device="cuda").transpose(2, 3)[:, 1]
    values = torch.full((pages, 2, 128, 1, 32), math.nan, dtype=torch.bfloat16, device="cuda").transpose(2, 3)[:, 0]
    keys.copy_(s.cache.keys)
    values.copy_(s.cache.values)
    assert keys.stride()[1:] == (64, 2048, 1) and values.stride()[1:] == (32, 32, 1)
    expected, tolerance, _, _ = s.exact(scales_of(1))
    got = da.paged_attention_hip(s.query, da.PagedCache(keys, values), *s.where()[2:], scales_of(1).cuda())
    close(got.cpu(), expected, tolerance)
