"""Performance cases of the language model's serving operators.

Four operators around a paged cache of routed keys and values, and the numbers
that a model answers with:

* ``append``: the new tokens' keys and values go into the cache's pages;
* ``attend``: a chunk of new tokens (one token, too) attends to its sequence's
  cached tokens, a score map for each temperature; with ``track``, every
  cached token's accumulated attention weight comes back as well;
* ``evict``: of each sequence the most recent tokens and those of the largest
  accumulated weight stay, and move into fresh pages;
* ``score``: log probabilities of given tokens, the distributions' entropies
  and the most probable alternatives; in training with the logits' gradient.

The cache is a pair of tensors: keys ``[pages, page_size, branches, R]``, and
values in tiles of 32 tokens, a feature's tokens side by side:
``[pages, page_size / 32, D, 32]``.  ``listed()`` holds the cases that are
reported, ``draw()`` more of the same ranges, ``run()`` one pass (in plain
32-bit torch, or with ``own`` through the framework), ``exact()`` the same
results in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_TILE = 32


def _attend(name: str, seqs: int, length: int, chunk: int, **options) -> dict:
    case = {"kind": "attend", "seqs": seqs, "length": length, "chunk": chunk, "ragged": True, "branches": 1, "maps": 1,
            "width": 256, "value": 512, "page": 64, "dtype": "bf16", "mix": False, "track": False, **options}
    return {"name": name, **case} if name else case


def _append(name: str, seqs: int, length: int, chunk: int, **options) -> dict:
    case = {"kind": "append", "seqs": seqs, "length": length, "chunk": chunk, "ragged": True, "branches": 1,
            "width": 256, "value": 512, "page": 64, "dtype": "bf16", **options}
    return {"name": name, **case} if name else case


def _evict(name: str, seqs: int, length: int, keep: int, recent: int, **options) -> dict:
    case = {"kind": "evict", "seqs": seqs, "length": length, "keep": keep, "recent": recent, "branches": 1,
            "width": 256, "value": 512, "page": 64, "dtype": "bf16", **options}
    return {"name": name, **case} if name else case


def _score(name: str, rows: int, vocab: int, **options) -> dict:
    case = {"kind": "score", "rows": rows, "vocab": vocab, "top": 0, "dtype": "bf16", "train": False, **options}
    return {"name": name, **case} if name else case


def listed() -> list[dict]:
    return [
        # The next token of one short conversation: latency counts.
        _attend("attend-token", 1, 500, 1),
        # A serving step of the default layer: many sequences, a token each.
        _attend("attend-batch", 64, 4096, 1),
        # One token against a very long context.
        _attend("attend-long", 1, 131072, 1, ragged=False),
        # Prompts that arrive in chunks behind what is cached already.
        _attend("attend-chunk", 4, 8192, 512, ragged=False),
        # Prompts and single tokens in one step, four maps mixed, the weights
        # kept for a later eviction, odd lengths everywhere.
        _attend("attend-mixed", 16, 2999, 201, branches=4, maps=4, width=128, dtype="fp16", mix=True, track=True),
        # One new token of each of many sequences into the pages.
        _append("append-step", 64, 700, 1),
        # Prompts' chunks into the pages, odd lengths, two branches.
        _append("append-chunk", 16, 1999, 777, branches=2, dtype="fp16"),
        # Conversations cut to half of their cache.
        _evict("evict-step", 8, 1001, 512, 64),
        # Long documents cut to a quarter, where the cache's bytes count.
        _evict("evict-long", 4, 32768, 8192, 1024, dtype="fp16"),
        # What the model of the benchmark answers for one position.
        _score("score-token", 1, 2048, top=5),
        # Prompt scoring over a wide odd vocabulary with 20 alternatives.
        _score("score-wide", 2048, 50001, top=20, dtype="fp16"),
        # A training step's loss over a long batch: forward and gradient.
        _score("score-train", 4096, 32000, train=True),
    ]


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    """One more case: sizes spread over their logarithm, the layers' layouts
    those of the presets, both 16-bit types."""

    kind = rng.choice(("attend", "attend", "attend", "attend", "append", "evict", "evict", "score", "score", "score"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "score":
        rows, vocab = _log_int(rng, 1, 8192), _log_int(rng, 200, 131072)
        rows = max(1, min(rows, 4096 * 32000 // vocab))
        train = rng.random() < 0.4
        return _score("", rows, vocab, top=0 if train else rng.choice((0, 1, 5, 20, 32)), dtype=dtype, train=train)
    branches, maps, width = rng.choice(((1, 1, 256), (1, 1, 256), (1, 1, 512), (2, 1, 256), (1, 2, 256), (2, 2, 256), (4, 4, 128)))
    value = rng.choice((512, 512, 512, 192, 320, 768, 1024))
    shape = {"branches": branches, "width": width, "value": value, "page": rng.choice((32, 64, 64, 128)), "dtype": dtype}
    row = branches * width + value
    if kind == "evict":
        length = _log_int(rng, 64, 32768)
        keep = max(1, int(length * rng.uniform(0.1, 0.9)))
        seqs = max(1, min(_log_int(rng, 1, 32), 4 * 32768 * 768 // (length * row)))
        return _evict("", seqs, length, keep, rng.randint(0, keep), **shape)
    if kind == "append":
        length = _log_int(rng, 1, 2000)
        chunk = min(length, _log_int(rng, 1, 1000))
        seqs = max(1, min(_log_int(rng, 1, 64), 16 * 1999 * 1024 // (length * row)))
        return _append("", seqs, length, chunk, ragged=rng.random() < 0.8, **shape)
    length = _log_int(rng, 1, 65536)
    chunk = 1 if rng.random() < 0.4 else min(length, _log_int(rng, 1, 1024))
    seqs = _log_int(rng, 1, 64)
    # No more cached bytes, and no more products, than the largest listed ones.
    seqs = max(1, min(seqs, 64 * 2560 * 768 // (length * row)))
    chunk = max(1, min(chunk, 4 * 512 * 5120 * 768 // (seqs * length * maps * (width * max(1, branches // maps) + value))))
    return _attend("", seqs, length, chunk, ragged=rng.random() < 0.8, maps=maps, mix=maps > 1 and rng.random() < 0.6,
                   track=rng.random() < 0.3, **shape)


def _sizes(case: dict) -> tuple[list[int], list[int]]:
    """``(lengths, chunks)`` of the sequences: the longest first, the others
    down to a quarter; new tokens from the chunk down to one, the last
    sequence of a larger batch without any."""

    seqs, chunk = case["seqs"], case.get("chunk", 0)
    lengths, chunks = [], []
    for i in range(seqs):
        part = i / seqs if case.get("ragged", True) else 0.0
        length = max(1, int(case["length"] * (1 - 0.75 * part)))
        new = max(1, int(chunk * (1 - part) ** 2))
        if chunk > 1 and part > 0 and i == seqs - 1 and seqs > 4:
            new = 0
        lengths.append(length)
        chunks.append(min(new, length))
    return lengths, chunks


def _unit_rows(*shape: int, center=None):
    """Routed rows: unit length, around a direction that they share."""

    rows = torch.randn(*shape)
    if center is not None:
        rows = rows + center
    return rows / rows.norm(dim=-1, keepdim=True)


def _pages(case: dict, lengths: list[int], spare: int) -> tuple[int, torch.Tensor]:
    """``(pages, table)``: a pool with a few pages more than the sequences
    need, which lie in it in no order; unused entries of the table are 0."""

    page = case["page"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages)
    table = torch.zeros(len(lengths), max(counts), dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n].int()
        at += n
    return pages, table


def prepare(case: dict, seed: int) -> dict:
    dtype = _DTYPES[case["dtype"]]
    torch.manual_seed(seed)
    state = {"case": case, "dtype": dtype}
    with torch.device("cuda"):
        if case["kind"] == "score":
            rows, vocab = case["rows"], case["vocab"]
            # A model's logits: a few tokens stand out in each row.
            logits = torch.randn(rows, vocab) * 2
            logits[torch.rand(rows, vocab) < 0.001] += 6
            state["logits"] = logits.to(dtype)
            state["tokens"] = torch.randint(0, vocab, (rows,))
            if case["train"]:
                # The loss: the mean negative log probability, and a little
                # of the entropy.
                state["grad"] = (torch.full((rows,), -1.0 / rows), torch.full((rows,), 0.01 / rows))
            return state
    lengths, chunks = _sizes(case)
    pages, table = _pages(case, lengths, 3)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
    state["table"] = table.cuda()
    with torch.device("cuda"):
        branches, width, value, page = case["branches"], case["width"], case["value"], case["page"]
        # Routed rows are held in fp16 beside values of the model's type.
        center = torch.randn(width) * 0.5
        state["keys"] = _unit_rows(pages, page, branches, width, center=center).half()
        state["values"] = torch.randn(pages, page // _TILE, value, _TILE).to(dtype)
        if case["kind"] == "evict":
            capacity = state["table"].shape[1] * page
            # Accumulated weights fall off steeply from a few heavy tokens.
            weights = torch.rand(len(lengths), capacity) ** 8
            weights[:, :4] += 2
            weights[:, 7::50] = 0.25   # equal ones
            state["weights"] = weights * (torch.arange(capacity)[None] < state["lengths"][:, None])
            kept = [min(n, case["keep"]) for n in lengths]
        else:
            offsets = [0]
            for n in chunks:
                offsets.append(offsets[-1] + n)
            state["chunks"], state["max_chunk"] = chunks, max(chunks)
            state["offsets"] = torch.tensor(offsets, dtype=torch.int32)
            if case["kind"] == "append":
                state["key"] = _unit_rows(offsets[-1], branches, width, center=center).half()
                state["value"] = torch.randn(offsets[-1], value).to(dtype)
            else:
                maps = case["maps"]
                state["query"] = _unit_rows(offsets[-1], branches, width, center=center).half()
                state["scales"] = 16.0 * torch.exp(torch.linspace(-0.2, 0.2, maps)) if maps > 1 else torch.full((1,), 16.0)
                state["mix"] = torch.softmax(torch.randn(maps), 0) if case["mix"] else None
                if case["track"]:
                    weights = torch.rand(len(lengths), state["table"].shape[1] * page)
                    state["weights"] = weights
    if case["kind"] == "evict":
        out_pages, out_table = _pages(case, kept, 1)
        with torch.device("cuda"):
            state["out_table"] = out_table.cuda()
            state["out_keys"] = torch.zeros(out_pages, page, branches, width, dtype=torch.float16)
            state["out_values"] = torch.zeros(out_pages, page // _TILE, value, _TILE, dtype=dtype)
    return state


# ---- plain forms, 32 bits ---------------------------------------------------


def _new_tokens(state: dict):
    """``(sequence, position, visible length)`` of each new token, on the GPU."""

    offsets, lengths = state["offsets"].long(), state["lengths"].long()
    total = sum(state["chunks"])
    n = torch.arange(total, device=offsets.device)
    seq = (n[:, None] >= offsets[None, 1:]).sum(1)
    position = lengths[seq] - (offsets[seq + 1] - n)
    return seq, position


def _slots(state: dict, seq, position):
    """``(page, slot)`` of the sequences' positions."""

    page = state["case"]["page"]
    return state["table"].long()[seq, position // page], position % page


def _cached_rows(state: dict):
    """The sequences' cached keys ``[B, capacity, H, R]`` and values
    ``[B, capacity, D]`` as 32-bit rows; positions behind a sequence are zero."""

    table = state["table"].long()
    keys = state["keys"][table].flatten(1, 2).float()
    values = state["values"][table].transpose(-1, -2).flatten(1, 3).float()
    behind = torch.arange(keys.shape[1], device=keys.device)[None] >= state["lengths"][:, None]
    return keys.masked_fill(behind[..., None, None], 0), values.masked_fill(behind[..., None], 0)


def _plain_attend(state: dict):
    case, dtype = state["case"], state["dtype"]
    branches, maps, width = case["branches"], case["maps"], case["width"]
    keys, values = _cached_rows(state)
    seq, position = _new_tokens(state)
    batch, capacity, chunk = len(state["chunks"]), keys.shape[1], state["max_chunk"]
    first = state["offsets"].long()[seq]
    place = torch.arange(len(seq), device=seq.device) - first
    # New tokens padded to [B, chunk], their heads as score maps.
    query = keys.new_zeros(batch, chunk, branches, width)
    query[seq, place] = state["query"].float()
    at = torch.full((batch, chunk), -1, device=seq.device)
    at[seq, place] = position
    factor = 1.0
    if branches > maps:
        factor = (branches // maps) ** -0.5
        query, keys = query.reshape(batch, chunk, maps, -1), keys.reshape(batch, capacity, maps, -1)
    elif maps > branches:
        query = query.repeat_interleave(maps // branches, dim=2)
        keys = keys.repeat_interleave(maps // branches, dim=2)
    scores = torch.matmul(query.transpose(1, 2).contiguous(), keys.permute(0, 2, 3, 1).contiguous())
    scores = scores * (state["scales"] * factor)[None, :, None, None]
    hidden = torch.arange(capacity, device=seq.device)[None, None] > at[:, :, None]
    scores = scores.masked_fill(hidden[:, None], float("-inf"))
    largest = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    probs = torch.exp(scores - largest)
    probs = probs / probs.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(probs, values[:, None]).transpose(1, 2)   # [B, chunk, S, D]
    out = out[seq, place]
    if state["mix"] is not None:
        out = (out * state["mix"][None, :, None]).sum(1)
    out = out.to(dtype)
    if not case["track"]:
        return out
    # Tokens that are new in this chunk start from nothing.
    old = state["lengths"] - (state["offsets"][1:] - state["offsets"][:-1])
    before = torch.arange(capacity, device=seq.device)[None] < old[:, None]
    weights = torch.where(before, state["weights"], 0.0) + probs.sum((1, 2))
    return {"out": out, "weights": weights}


def _plain_append(state: dict):
    seq, position = _new_tokens(state)
    page, slot = _slots(state, seq, position)
    state["keys"][page, slot] = state["key"]
    state["values"][page, slot // _TILE, :, slot % _TILE] = state["value"]
    return {"keys": state["keys"], "values": state["values"]}


def _plain_evict(state: dict):
    case = state["case"]
    keep, page = case["keep"], case["page"]
    weights, lengths = state["weights"], state["lengths"].long()
    batch, capacity = weights.shape
    index = torch.arange(capacity, device=weights.device)[None]
    counts = lengths.clamp_max(keep)
    # Candidates behind the most recent tokens, the heaviest first and equal
    # ones in order; recent tokens come before all, others never.
    rank = torch.where(index < lengths[:, None], weights, float("-inf"))
    rank = torch.where((index >= (lengths - min(case["recent"], keep))[:, None]) & (index < lengths[:, None]), float("inf"), rank)
    chosen = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :keep]
    slots = torch.arange(chosen.shape[1], device=weights.device)[None]
    chosen = torch.where(slots < counts[:, None], chosen, capacity)
    chosen = torch.sort(chosen, dim=1).values
    valid = slots < counts[:, None]
    kept = torch.full((batch, keep), -1, dtype=torch.int32, device=weights.device)
    kept[:, :chosen.shape[1]] = torch.where(valid, chosen, -1).int()
    seq, place = torch.nonzero(valid, as_tuple=True)
    source = chosen[seq, place]
    from_page, from_slot = _slots(state, seq, source)
    to_page, to_slot = state["out_table"].long()[seq, place // page], place % page
    state["out_keys"][to_page, to_slot] = state["keys"][from_page, from_slot]
    state["out_values"][to_page, to_slot // _TILE, :, to_slot % _TILE] = state["values"][from_page, from_slot // _TILE, :, from_slot % _TILE]
    moved = weights.new_zeros(batch, state["out_table"].shape[1] * page)
    moved[seq, place] = weights[seq, source]
    return {"kept": kept, "counts": counts.int(), "keys": state["out_keys"], "values": state["out_values"], "weights": moved}


def _plain_score(state: dict):
    case, tokens = state["case"], state["tokens"]
    x = state["logits"].float()
    largest = x.amax(-1, keepdim=True)
    shifted = x - largest
    weights = torch.exp(shifted)
    total = weights.sum(-1, keepdim=True)
    logs = shifted - torch.log(total)
    probs = weights / total
    chosen = logs.gather(1, tokens[:, None])[:, 0]
    entropy = -(probs * logs).sum(-1)
    out = {"log_probs": chosen, "entropy": entropy}
    if case["top"]:
        index = torch.arange(x.shape[1], device=x.device)
        left, tops = x.clone(), []
        for _ in range(case["top"]):
            best = left.amax(-1, keepdim=True)
            first = torch.where(left == best, index, x.shape[1]).amin(-1, keepdim=True)
            left.scatter_(1, first, float("-inf"))
            tops.append(first)
        out["top_tokens"] = torch.cat(tops, 1)
        out["top_log_probs"] = logs.gather(1, out["top_tokens"])
    if case["train"]:
        at_token, at_entropy = state["grad"]
        grad = -probs * (at_token[:, None] + at_entropy[:, None] * (logs + entropy[:, None]))
        grad.scatter_add_(1, tokens[:, None], at_token[:, None])
        out["grad"] = grad.to(state["dtype"])
    return out


# ---- the framework's calls --------------------------------------------------


def _package():
    at = os.path.join(_ROOT, "double-attention_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import double_attention

    return double_attention


def _own(state: dict):
    da = _package()
    case = state["case"]
    kind = case["kind"]
    if kind == "score":
        if not case["train"]:
            got = da.token_log_probs_hip(state["logits"], state["tokens"], top=case["top"])
            out = {"log_probs": got.log_probs, "entropy": got.entropy}
            if case["top"]:
                out["top_tokens"], out["top_log_probs"] = got.top_tokens, got.top_log_probs
            return out
        logits = state["logits"].detach().requires_grad_()
        got = da.token_log_probs_hip(logits, state["tokens"])
        (grad,) = torch.autograd.grad((got.log_probs, got.entropy), logits, state["grad"])
        return {"log_probs": got.log_probs.detach(), "entropy": got.entropy.detach(), "grad": grad}
    cache = da.PagedCache(state["keys"], state["values"])
    if kind == "append":
        da.cache_append_hip(cache, state["key"], state["value"], state["table"], state["lengths"], state["offsets"],
                            max_chunk=state["max_chunk"])
        return {"keys": state["keys"], "values": state["values"]}
    if kind == "evict":
        kept, counts = da.cache_select_hip(state["weights"], state["lengths"], case["keep"], case["recent"])
        out = da.PagedCache(state["out_keys"], state["out_values"])
        weights = da.cache_compact_hip(cache, state["table"], kept, counts, out, state["out_table"], weights=state["weights"])
        return {"kept": kept, "counts": counts, "keys": state["out_keys"], "values": state["out_values"], "weights": weights}
    where = (state["query"], cache, state["table"], state["lengths"], state["offsets"], state["scales"])
    if not case["track"]:
        return da.paged_attention_hip(*where, mix=state["mix"], max_chunk=state["max_chunk"])
    out, weights = da.paged_attention_weights_hip(*where, weights=state["weights"], mix=state["mix"], max_chunk=state["max_chunk"])
    return {"out": out, "weights": weights}


def run(state: dict):
    return _own(state) if own else _plain(state)


def _plain(state: dict):
    return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict, "score": _plain_score}[state["case"]["kind"]](state)


def work(case: dict) -> dict:
    if case["kind"] == "score":
        cells, top = case["rows"] * case["vocab"], case["top"]
        # Logits read once; in training their gradient written.
        return {"bytes": 2 * cells * (2 if case["train"] else 1) + case["rows"] * (16 + 12 * top),
                "flops": cells * (12 if case["train"] else 6)}
    lengths, chunks = _sizes(case)
    key, value = case["branches"] * case["width"], case["value"]
    if case["kind"] == "append":
        return {"bytes": 4 * sum(chunks) * (key + value), "flops": 0}
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        # Every weight read, the kept tokens' rows and weights moved.
        return {"bytes": 4 * sum(lengths) + 4 * kept * (key + value) + 12 * kept, "flops": 0}
    maps = case["maps"]
    seen = sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, chunks))
    read = sum(n for n, c in zip(lengths, chunks) if c)
    out = sum(chunks) * value * (1 if case["mix"] else maps)
    tracked = 8 * sum(lengths) if case["track"] else 0
    return {"bytes": 2 * read * (key + value) + 2 * sum(chunks) * key + 2 * out + tracked,
            "flops": 2 * seen * (max(key, maps * case["width"]) + maps * value)}


# ---- the same results in 64 bits --------------------------------------------


def _exact_attend(state: dict):
    case = state["case"]
    maps, branches, page = case["maps"], case["branches"], case["page"]
    lengths, chunks = _sizes(case)
    outs, sums = [], torch.zeros(len(lengths), state["table"].shape[1] * page, dtype=torch.float64, device="cuda")
    start = 0
    for b, (length, new) in enumerate(zip(lengths, chunks)):
        used = state["table"][b, :-(-length // page)].long()
        keys = state["keys"][used].reshape(-1, branches, case["width"])[:length].double()
        values = state["values"][used].transpose(2, 3).reshape(-1, case["value"])[:length].double()
        if case["track"]:
            sums[b, :length - new] = state["weights"][b, :length - new].double()
        if new == 0:
            continue
        query = state["query"][start:start + new].double()
        start += new
        places = torch.arange(length, device="cuda")
        seen = places[None] <= torch.arange(length - new, length, device="cuda")[:, None]
        per_map = []
        for s in range(maps):
            if branches >= maps:
                mine = range(s * (branches // maps), (s + 1) * (branches // maps))
            else:
                mine = [s // (maps // branches)]
            scores = sum(torch.mm(query[:, h], keys[:, h].t()) for h in mine) / math.sqrt(len(mine))
            scores = torch.where(seen, scores * state["scales"][s].double(), torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
            probs = torch.softmax(scores, -1)
            if case["track"]:
                sums[b, :length] += probs.sum(0)
            per_map.append(torch.mm(probs, values))
        if case["mix"]:
            outs.append(sum(w * o for w, o in zip(state["mix"].double(), per_map)))
        else:
            outs.append(torch.stack(per_map, 1))
    out = torch.cat(outs)
    return {"out": out, "weights": sums} if case["track"] else out


def _exact_score(state: dict):
    case = state["case"]
    x = state["logits"].double().requires_grad_(case["train"])
    logs = torch.log_softmax(x, -1)
    chosen = logs[torch.arange(case["rows"], device="cuda"), state["tokens"]]
    entropy = -(torch.exp(logs) * logs).sum(-1)
    out = {"log_probs": chosen.detach(), "entropy": entropy.detach()}
    if case["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_tokens"], out["top_log_probs"] = order, logs.gather(1, order)
    if case["train"]:
        both = [g.double() for g in state["grad"]]
        (out["grad"],) = torch.autograd.grad((chosen, entropy), x, both)
    return out


def _exact_append(state: dict):
    case = state["case"]
    keys, values, page, start = state["keys"].double(), state["values"].double(), case["page"], 0
    for b, (length, new) in enumerate(zip(*_sizes(case))):
        at = torch.arange(length - new, length, device="cuda")
        pages, slots = state["table"][b].long()[at // page], at % page
        keys[pages, slots] = state["key"][start:start + new].double()
        values[pages, slots // _TILE, :, slots % _TILE] = state["value"][start:start + new].double()
        start += new
    return {"keys": keys, "values": values}


def _exact_evict(state: dict):
    case = state["case"]
    page, lengths = case["page"], _sizes(case)[0]
    keys, values = state["out_keys"].double(), state["out_values"].double()
    kept = torch.full((len(lengths), case["keep"]), -1, dtype=torch.int32, device="cuda")
    moved = torch.zeros(len(lengths), state["out_table"].shape[1] * page, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lengths):
        count = min(length, case["keep"])
        recent = min(case["recent"], count)
        order = torch.sort(state["weights"][b, :length - recent], descending=True, stable=True).indices[:count - recent]
        chosen = torch.cat((torch.sort(order).values, torch.arange(length - recent, length, device="cuda")))
        kept[b, :count] = chosen.int()
        moved[b, :count] = state["weights"][b, chosen].double()
        to = torch.arange(count, device="cuda")
        source, target = state["table"][b].long()[chosen // page], state["out_table"][b].long()[to // page]
        keys[target, to % page] = state["keys"][source, chosen % page].double()
        taken = state["values"][source, chosen % page // _TILE, :, chosen % _TILE].double()
        values[target, to % page // _TILE, :, to % _TILE] = taken
    counts = torch.tensor([min(n, case["keep"]) for n in lengths], dtype=torch.int32, device="cuda")
    return {"kept": kept, "counts": counts, "keys": keys, "values": values, "weights": moved}


def exact(case: dict, seed: int):
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict, "score": _exact_score}[case["kind"]](prepare(case, seed))
