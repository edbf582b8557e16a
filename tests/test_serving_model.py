"""The language model over paged caches: cached and whole forwards, eviction,
steps captured in graphs, and the log probabilities of next tokens."""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

import double_attention as da

CONFIGS = {
    "one-map": dict(),
    "two-branches": dict(qk_branches=2, outer_maps=1),
    "two-maps": dict(qk_branches=1, outer_maps=2),
    "four-maps": dict(qk_branches=4, outer_maps=4, routing_dim=64),
    "concat": dict(qk_branches=2, outer_maps=2, map_combine="concat"),
    "no-projection": dict(qk_branches=2, outer_maps=2, output_projection=False, value_bias=False),
    "no-norms": dict(normalize_routing_input=False, normalize_routing_output=False),
    "query-feedforward": dict(q_dictionary_feedforward=True, dictionary_size=96),
    "tied": dict(untied_dictionary=False, learnable_beta=True),
}


def model_of(name: str = "one-map", dtype: torch.dtype = torch.bfloat16, layers: int = 2, **options) -> da.DoubleAttentionLM:
    torch.manual_seed(3)
    config = da.DoubleAttentionConfig(
        **{"model_dim": 128, "routing_dim": 128, "dictionary_size": 64, "initial_score_scale": 8.0, "backend": "hip", **CONFIGS[name]}
    )
    model = da.DoubleAttentionLM(97, 200, config, layers, feedforward_dim=96, **options)
    return model.to(dtype).eval()


def whole_logits(model: da.DoubleAttentionLM, tokens: torch.Tensor) -> torch.Tensor:
    """Logits of the plain composition in fp64, on the host, with the model's rounded parameters."""

    plain = copy.deepcopy(model).cpu().double()
    for block in plain.stack.blocks:
        block.attention.config = block.attention.config.with_updates(backend="torch")
    plain.stack.config = plain.stack.config.with_updates(backend="torch")
    with torch.no_grad():
        return plain(tokens.cpu())[0]


def rms(t: torch.Tensor) -> float:
    return float(t.double().pow(2).mean().sqrt())


def ids(*counts: int, seed: int = 0) -> list[torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 97, (n,), generator=g) for n in counts]


# ---- refusals ---------------------------------------------------------------


def test_refusals_of_the_sequences() -> None:
    model = model_of()
    with pytest.raises(ValueError, match="at least one sequence"):
        da.CachedSequences(model, 0, 4)
    with pytest.raises(NotImplementedError, match="page sizes"):
        da.CachedSequences(model, 1, 4, page_size=48)
    s = da.CachedSequences(model, 2, 3, page_size=32)
    tokens = ids(5)[0]
    for counts in ([5], [6, -1], [1, 1, 3]):
        with pytest.raises(ValueError, match="counts"):
            s.extend(tokens, counts)
    with pytest.raises(ValueError, match="int64"):
        s.extend(tokens, [3, 3])
    with pytest.raises(ValueError, match="int64"):
        s.extend(tokens.int(), [3, 2])
    with pytest.raises(ValueError, match="positions"):
        s.extend(ids(201)[0], [201, 0])
    for bad in (97, -1):
        with pytest.raises(ValueError, match="must be in"):
            s.extend(torch.tensor([1, bad]), [1, 1])
    with pytest.raises(RuntimeError, match="does not fit"):
        s.extend(ids(97)[0], [97, 0])
    with pytest.raises(RuntimeError, match="more pages"):
        s.extend(ids(98)[0], [65, 33])
    with pytest.raises(RuntimeError, match="gather_weights"):
        s.evict(4)
    with pytest.raises(RuntimeError):   # no kernels for a model on the host
        s.extend(tokens, [3, 2])
    assert s.free_pages == 3 and s.lengths == [0, 0] and s.positions == [0, 0]
    s = da.CachedSequences(model, 2, 3, page_size=32, gather_weights=True)
    for keep, recent in ((0, 0), (3, 4), (3, -1)):
        with pytest.raises(ValueError, match="evict"):
            s.evict(keep, recent)
    s.evict(3)   # nothing to cut


def test_refusals_of_the_model() -> None:
    model = model_of()
    caches = model.paged_caches(2, 32)
    assert len(caches) == 2 and caches[0].keys.dtype is torch.float16 and caches[0].values.dtype is torch.bfloat16
    assert model_of(dtype=torch.float16).paged_caches(2)[0].values.dtype is torch.float16
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    offsets = torch.tensor([0, 1], dtype=torch.int32)
    token = torch.zeros(1, dtype=torch.int64)
    where = (caches, table, lengths, offsets)
    with pytest.raises(ValueError, match=r"shape \[N\]"):
        model.cached_forward(token[None], token[None], *where)
    with pytest.raises(ValueError, match=r"shape \[N\]"):
        model.cached_forward(token, token[:0], *where)
    with pytest.raises(ValueError, match="2 caches"):
        model.cached_forward(token, token, caches[:1], *where[1:])
    with pytest.raises(RuntimeError):
        model.cached_forward(token, token, *where)
    with pytest.raises(NotImplementedError, match="fp16 and bf16"):
        model_of(dtype=torch.float32).cached_forward(token, token, *where)
    loose = model_of()
    loose.stack.config = loose.stack.config.with_updates(causal=False)
    with pytest.raises(ValueError, match="causal"):
        loose.cached_forward(token, token, *where)
    with pytest.raises(ValueError, match="ROCm device"):
        plain = model_of(dtype=torch.float32)
        for block in plain.stack.blocks:
            block.attention.config = block.attention.config.with_updates(backend="torch")
        plain.stack.config = plain.stack.config.with_updates(backend="torch")
        plain.token_log_probs(torch.zeros(1, 3, dtype=torch.int64))


# ---- cached and whole forwards ---------------------------------------------


def check_cached(model: da.DoubleAttentionLM, chunks: list[list[int]], page_size: int = 32) -> None:
    """Both forwards round the same values at the same places and differ in the
    order of their fp32 sums: their errors against fp64 have one distribution.
    Over some thousands of logits the ratio of two root mean squares of such
    errors (a few layers' correlated roundings) stays well inside 1.5."""

    counts = [sum(c) for c in zip(*chunks)]
    tokens = ids(*counts, seed=len(chunks))
    total = sum(counts)
    pages = sum(-(-n // page_size) for n in counts)
    s = da.CachedSequences(model, len(counts), pages, page_size=page_size)
    got = [[] for _ in counts]
    done = [0] * len(counts)
    for chunk in chunks:
        packed = torch.cat([t[at:at + n] for t, at, n in zip(tokens, done, chunk)])
        logits = s.extend(packed, chunk)
        for b, part in enumerate(logits.split(chunk)):
            got[b].append(part)
            done[b] += chunk[b]
    assert s.lengths == counts and s.free_pages == 0
    cached = torch.cat([torch.cat(parts) for parts in got]).cpu()
    with torch.no_grad():
        whole = torch.cat([model(t[None].cuda())[0][0] for t in tokens if len(t)]).cpu()
    expected = torch.cat([whole_logits(model, t[None])[0] for t in tokens if len(t)])
    assert cached.shape == (total, 97)
    assert rms(cached - expected) <= 1.5 * rms(whole - expected)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("name", CONFIGS)
def test_cached_forward_is_the_whole_one(name, dtype) -> None:
    check_cached(model_of(name, dtype).cuda(), [[33, 0, 64], [1, 1, 31], [40, 1, 1], [1, 1, 1]])


@pytest.mark.gpu
@pytest.mark.parametrize("options", [dict(norm="rms"), dict(dictionary_group_size=1)], ids=["rms", "two-banks"])
def test_cached_forward_of_other_models(options) -> None:
    check_cached(model_of(**options).cuda(), [[150, 3], [1, 1], [49, 7]], page_size=64)


@pytest.mark.gpu
def test_cached_forward_on_8_bit_feedforward() -> None:
    # The 8-bit rounding of the activations dwarfs the 16-bit ones, and is the same in both.
    model = model_of(norm="rms").cuda()
    model.stack.quantize_feedforward()
    check_cached(model, [[70, 20], [1, 1], [5, 0]])


@pytest.mark.gpu
def test_one_token_at_a_time_and_last_rows() -> None:
    model = model_of("two-maps").cuda()
    check_cached(model, [[1, 1]] * 40)
    s = da.CachedSequences(model, 3, 8, page_size=32)
    tokens = torch.cat(ids(5, 0, 7))
    everything = s.extend(tokens, [5, 0, 7])
    for b in range(3):
        s.release(b)
    assert s.free_pages == 8
    last = s.extend(tokens, [5, 0, 7], last_only=True)
    # One row's logits come from a library product of another height.
    assert last.shape == (2, 97)
    torch.testing.assert_close(last, everything[[4, 11]], rtol=2 ** -7, atol=2 ** -7 * rms(everything))
    assert s.extend(tokens[:0], [0, 0, 0]).shape == (0, 97)


@pytest.mark.gpu
def test_eviction_of_a_model_s_sequences() -> None:
    model = model_of("two-maps").cuda()
    s = da.CachedSequences(model, 3, 16, page_size=32, gather_weights=True)
    counts = [100, 20, 70]
    s.extend(torch.cat(ids(*counts)), counts)
    s.extend(torch.cat(ids(1, 1, 1, seed=1)), [1, 1, 1])
    lengths = list(s.lengths)
    assert lengths == [101, 21, 71]
    before = [[c.rows(s.pages(b), n) for b, n in enumerate(lengths)] for c in s.caches]
    weights = s.weights.cpu()
    for b, n in enumerate(lengths):
        # A row gives its visible tokens one, in each of two maps: sums of fp32
        # probabilities, up to their roundings (n * 2^-24 each).
        torch.testing.assert_close(weights[:, b].sum(-1), torch.full((2,), 2.0 * n), rtol=n * 2 ** -22, atol=0)
        assert not weights[:, b, n:].any()
    free = s.free_pages
    s.evict(40, 8)
    assert s.lengths == [40, 21, 40] and s.positions == lengths
    assert s.free_pages == free + (4 - 2) + (3 - 2)
    for layer, cache in enumerate(s.caches):
        for b, n in enumerate(lengths):
            kept = torch.arange(n)
            if n > 40:
                heavy = torch.sort(weights[layer, b, :n - 8], descending=True, stable=True).indices[:32]
                kept = torch.cat((heavy.sort().values, torch.arange(n - 8, n)))
            keys, values = cache.rows(s.pages(b), len(kept))
            assert torch.equal(keys, before[layer][b][0][kept.cuda()]) and torch.equal(values, before[layer][b][1][kept.cuda()])
            assert torch.equal(s.weights[layer, b].cpu()[:len(kept)], weights[layer, b, kept])
            assert not s.weights[layer, b, len(kept):].any()
    # The next token attends to what stayed: as over a cache that never held more.
    tokens = torch.cat(ids(2, 2, 2, seed=2))
    other = da.CachedSequences(model, 3, 16, page_size=32)
    other._pages, other._free = [[3, 4], [0, 9], [7, 8]], [1, 2, 5, 6, 10, 11, 12, 13, 14, 15]
    other.lengths, other.positions = list(s.lengths), list(s.positions)
    for mine, theirs in zip(other.caches, s.caches):
        for b in range(3):
            to, of = other.pages(b), s.pages(b)
            mine.keys[to[:len(of)]] = theirs.keys[of]
            mine.values[to[:len(of)]] = theirs.values[of]
    torch.testing.assert_close(s.extend(tokens, [2, 2, 2]), other.extend(tokens, [2, 2, 2]), rtol=0, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("made_in,used_in", [(True, False), (False, True), (True, True)])
def test_sequences_in_inference_mode(made_in, used_in) -> None:
    model = model_of().cuda()
    expected = None
    for made, used in ((False, False), (made_in, used_in)):
        with torch.inference_mode(made):
            s = da.CachedSequences(model, 2, 8, page_size=32, gather_weights=True)
        with torch.inference_mode(used):
            s.extend(torch.cat(ids(40, 9)), [40, 9])
            s.evict(20, 4)
            s.extend(torch.cat(ids(1, 2, seed=1)), [1, 2])
            s.release(1)
            logits = s.extend(torch.cat(ids(3, 5, seed=2)), [3, 5])
        assert s.lengths == [24, 5] and s.positions == [44, 5]
        if expected is None:
            expected = logits
    assert torch.equal(logits, expected)


@pytest.mark.gpu
def test_sequences_that_wait_or_start_anew() -> None:
    model = model_of().cuda()
    s = da.CachedSequences(model, 2, 8, page_size=32, gather_weights=True)
    s.extend(torch.cat(ids(40, 33)), [40, 33])
    before = s.weights.clone()
    s.extend(ids(3, seed=1)[0], [3, 0])
    assert torch.equal(s.weights[:, 1], before[:, 1]) and not torch.equal(s.weights[:, 0], before[:, 0])
    s.release(0)
    alone = da.CachedSequences(model, 2, 8, page_size=32, gather_weights=True)
    alone.extend(torch.cat(ids(0, 33)), [0, 33])
    again = [t.extend(ids(35, seed=2)[0], [35, 0]) for t in (s, alone)]
    assert torch.equal(*again) and torch.equal(s.weights[:, 0], alone.weights[:, 0])


@pytest.mark.gpu
def test_decoding_step_as_a_graph() -> None:
    model = model_of("two-branches").cuda()
    page, sequences, steps = 32, 3, 5
    s = da.CachedSequences(model, sequences, 12, page_size=page, gather_weights=True)
    s.extend(torch.cat(ids(29, 64, 1)), [29, 64, 1])
    start = torch.tensor(s.lengths, dtype=torch.int32, device="cuda")
    table = torch.full((sequences, 4), -1, dtype=torch.int32)
    spare = iter(set(range(12)) - set(s.pages(0).tolist() + s.pages(1).tolist() + s.pages(2).tolist()))
    for b in range(sequences):
        own = s.pages(b).tolist()
        table[b, :len(own) + 1] = torch.tensor(own + [next(spare)])
    table = table.cuda()
    offsets = torch.arange(sequences + 1, dtype=torch.int32, device="cuda")

    def decode(caches, weights):
        token, lengths = torch.zeros(sequences, dtype=torch.int64, device="cuda"), start.clone()

        def step():
            lengths.add_(1)
            logits = model.cached_forward(token, lengths.long() - 1, caches, table, lengths, offsets, weights=weights, max_chunk=1,
                                          max_length=4 * page)
            best = da.token_log_probs_hip(logits, token, top=2)
            token.copy_(best.top_tokens[:, 0])
            return logits, best.top_log_probs

        return step, token, lengths

    def copies():
        return [da.PagedCache(c.keys.clone(), c.values.clone()) for c in s.caches], s.weights[:, :, :4 * page].contiguous()

    eager_caches, eager_weights = copies()
    eager, _, _ = decode(eager_caches, eager_weights)
    caches, weights = copies()
    step, token, lengths = decode(caches, weights)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    # Back to the start, then replayed beside the eager steps.
    token.zero_()
    lengths.copy_(start)
    for mine, kept in zip(caches, s.caches):
        mine.keys.copy_(kept.keys)
        mine.values.copy_(kept.values)
    weights.copy_(s.weights[:, :, :4 * page])
    for _ in range(steps):
        expected = eager()
        torch.cuda.synchronize()
        graph.replay()
        for got, want in zip(captured, expected):
            assert torch.equal(got, want)
        assert torch.equal(weights, eager_weights)


@pytest.mark.gpu
def test_linear_into_a_given_tensor() -> None:
    from double_attention.hip_ops import linear_hip

    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(128, 128, generator=g).cuda().bfloat16() for _ in range(2))
    both = torch.zeros(3, 128, 128, dtype=torch.bfloat16, device="cuda")
    assert linear_hip(x, w, out=both[1]).data_ptr() == both[1].data_ptr()
    assert torch.equal(both[1], linear_hip(x, w)) and not both[::2].any()
    assert torch.equal(linear_hip(x, w, activation="gelu", residual=x, out=both[0]), linear_hip(x, w, activation="gelu", residual=x))
    wide = torch.empty(128, 256, dtype=torch.bfloat16, device="cuda")
    for out in (both, both[0].float(), wide[:, :128], both.flatten()[4:4 + 128 * 128].view(128, 128), both[0].cpu()):
        with pytest.raises(ValueError, match="out must have"):
            linear_hip(x, w, out=out)
    for out in (x, w):
        with pytest.raises(ValueError, match="overlap"):
            linear_hip(x, w, out=out)
    with pytest.raises(ValueError, match="overlap"):
        linear_hip(x, w, residual=both[2], out=both[2])


# ---- log probabilities of next tokens --------------------------------------


@pytest.mark.gpu
def test_log_probs_of_next_tokens() -> None:
    model = model_of().cuda()
    tokens = torch.stack(ids(30, 30)).cuda()
    with torch.no_grad():
        logits = model(tokens)[0].double()
        result = model.token_log_probs(tokens, top=3, entropy=True)
    expected = torch.log_softmax(logits[:, :-1], -1)
    # fp32 statistics of some 100 logits of a few units.
    close = dict(rtol=2 ** -18, atol=2 ** -18)
    torch.testing.assert_close(result.log_probs.double(), expected.gather(-1, tokens[:, 1:, None])[..., 0], **close)
    torch.testing.assert_close(result.entropy.double(), -(expected.exp() * expected).sum(-1), **close)
    torch.testing.assert_close(result.top_log_probs.double(), expected.topk(3, -1).values, **close)
    assert result.top_tokens.shape == (2, 29, 3)


@pytest.mark.gpu
def test_training_on_log_probs_of_next_tokens() -> None:
    # The mean of -log p is the model's loss: its gradients differ by the
    # roundings of the logits' gradient (bf16, one half step of 2^-8 a value).
    model = model_of().cuda().train()
    tokens = torch.stack(ids(30, 30)).cuda()
    loss = -model.token_log_probs(tokens).log_probs.mean()
    grads = torch.autograd.grad(loss, list(model.parameters()), allow_unused=True)
    logits, _ = model(tokens)
    other = F.cross_entropy(logits[:, :-1].flatten(0, 1).float(), tokens[:, 1:].flatten())
    expected = torch.autograd.grad(other, list(model.parameters()), allow_unused=True)
    torch.testing.assert_close(loss, other, rtol=2 ** -18, atol=0)
    for (name, _), got, want in zip(model.named_parameters(), grads, expected):
        assert (got is None) == (want is None), name
        if got is not None and rms(want) > 1e-7:
            assert rms(got.double() - want.double()) <= 2 ** -6 * rms(want), name
