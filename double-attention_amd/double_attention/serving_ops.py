"""Serving operators of the language model on the gfx950 kernels.

* ``PagedCache``, ``paged_cache`` and ``cache_append_hip``: routed keys and
  values of cached tokens in pages, and new tokens into them;
* ``paged_attention_hip`` and ``paged_attention_weights_hip``: the outer
  attention of new tokens (a chunk of each sequence, or one token) over its
  cached tokens, and the weight that every cached token gathered;
* ``cache_select_hip`` and ``cache_compact_hip``: which tokens stay when
  sequences are cut, by their gathered weight, and their move into other pages;
* ``token_log_probs_hip``: log probabilities of given tokens, entropies and the
  most probable alternatives.

As in ``hip_ops``, PyTorch supplies memory and the current stream, and nothing
falls back to another implementation: a call the kernels do not cover raises.
``token_log_probs_hip`` is differentiable in the logits; the other calls refuse
tensors whose gradients autograd would record.  Page tables, lengths and offsets
are int32 tensors on the device and are not read on the host, so calls can be
captured in graphs.  The kernels run on the inputs' device, whichever is current.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from .hip_ops import routed_score_layout
from .int8_ops import _CODES, _FLOAT32, _HALF_CODES, _has_tangent, _launch, _no_grad

CACHE_TILE = 32             # tokens of a tile of values; page sizes are multiples of it
MAX_PAGE_SIZE = 4096
MAX_KEY_WIDTH = 1024
MAX_VALUE_DIM = 4096
MAX_MAPS = 64
MAX_TOP = _lib.MAX_TOP


class PagedCache(NamedTuple):
    """Cached tokens of one layer in pages of ``page_size`` tokens.

    ``keys``: ``[pages, page_size, branches, routing_dim]``, the routed key
    rows.  ``values``: ``[pages, page_size / 32, value_dim, 32]``, tiles of 32
    tokens with a feature's tokens side by side (what the attention's matrix
    instructions read).  A page is contiguous; the pages may lie further apart
    (a layer's part of a larger tensor).  Which pages are whose, a page table
    says: int32 ``[sequences, entries]``, a sequence's pages in order.
    """

    keys: Tensor
    values: Tensor

    @property
    def page_size(self) -> int:
        return self.keys.shape[1]

    def rows(self, pages: Tensor, length: int) -> tuple[Tensor, Tensor]:
        """Keys ``[length, branches, routing_dim]`` and values ``[length, value_dim]``
        of the first tokens of a sequence with these pages, in order (copies)."""

        pages = pages.long()
        keys = self.keys[pages].flatten(0, 1)[:length]
        values = self.values[pages].transpose(-1, -2).flatten(0, 2)[:length]
        return keys, values


def paged_cache(
    pages: int,
    page_size: int,
    branches: int,
    routing_dim: int,
    value_dim: int,
    *,
    key_dtype: torch.dtype = torch.float16,
    dtype: torch.dtype = torch.bfloat16,
    device: torch.device | str | None = None,
) -> PagedCache:
    """An empty cache.  ``key_dtype``: of the routed rows (fp16, or with bf16 values bf16)."""

    _check_sizes("paged_cache", pages, page_size, branches * routing_dim, value_dim)
    if (key_dtype, dtype) not in _TYPES:
        raise ValueError(f"paged_cache: keys of {key_dtype} beside values of {dtype}")
    keys = torch.zeros(pages, page_size, branches, routing_dim, dtype=key_dtype, device=device)
    return PagedCache(keys, torch.zeros(pages, page_size // CACHE_TILE, value_dim, CACHE_TILE, dtype=dtype, device=device))


_INT32, _INT64 = torch.int32, torch.int64
_TYPES = {(torch.float16, torch.float16), (torch.float16, torch.bfloat16), (torch.bfloat16, torch.bfloat16)}


def _check_sizes(what: str, pages: int, page_size: int, width: int, value_dim: int) -> None:
    if pages < 1:
        raise ValueError(f"{what}: a cache has at least one page")
    if page_size < CACHE_TILE or page_size % CACHE_TILE or page_size > MAX_PAGE_SIZE:
        raise NotImplementedError(f"{what}: page sizes are multiples of {CACHE_TILE} up to {MAX_PAGE_SIZE}, not {page_size}")
    if width < 64 or width % 64 or width > MAX_KEY_WIDTH:
        raise NotImplementedError(f"{what}: branches * routing_dim is a multiple of 64 up to {MAX_KEY_WIDTH}, not {width}")
    if value_dim < 64 or value_dim % 64 or value_dim > MAX_VALUE_DIM:
        raise NotImplementedError(f"{what}: value_dim is a multiple of 64 up to {MAX_VALUE_DIM}, not {value_dim}")


def _check_cache(what: str, cache: PagedCache) -> torch.device:
    keys, values = cache
    key_shape, value_shape = keys.shape, values.shape
    if len(key_shape) != 4 or len(value_shape) != 4 or value_shape[3] != CACHE_TILE or key_shape[0] != value_shape[0] or (
        key_shape[1] != value_shape[1] * CACHE_TILE
    ):
        raise ValueError(f"{what}: a cache is keys [pages, page_size, branches, R] and values [pages, page_size / {CACHE_TILE}, "
                         f"D, {CACHE_TILE}], got {tuple(key_shape)} and {tuple(value_shape)}")
    if (keys.dtype, values.dtype) not in _TYPES:
        raise ValueError(f"{what}: keys of {keys.dtype} beside values of {values.dtype}")
    if not keys.is_cuda:
        raise ValueError(f"{what}: HIP kernels require tensors on a ROCm device")
    if values.get_device() != keys.get_device():
        raise ValueError(f"{what}: all tensors must be on {keys.device}, got one on {values.device}")
    pages, page_size, branches, routing_dim = key_shape
    _check_sizes(what, pages, page_size, branches * routing_dim, value_shape[2])
    if not (keys.is_contiguous() and values.is_contiguous()) and (
        keys.stride()[1:] != (branches * routing_dim, routing_dim, 1)
        or values.stride()[1:] != (value_shape[2] * CACHE_TILE, CACHE_TILE, 1)
    ) and not (keys[0].is_contiguous() and values[0].is_contiguous()):   # (dimensions of size one have any stride)
        raise ValueError(f"{what}: a cache's pages are contiguous")
    return keys.device


def _check_int32(what: str, name: str, t: Tensor, shape: tuple[int, ...], device: torch.device) -> Tensor:
    if t.dtype is not _INT32 or t.shape != shape:
        raise ValueError(f"{what}: {name} is int32 of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device.index:
        raise ValueError(f"{what}: all tensors must be on {device}, got {name} on {t.device}")
    return t.contiguous()


def _cache_args(what: str, cache: PagedCache, page_table: Tensor, device: torch.device) -> tuple[_lib.PagedCacheArgs, Tensor]:
    """The C description of the cache, and the table that it points to."""

    if page_table.dtype is not _INT32 or page_table.ndim != 2:
        raise ValueError(f"{what}: page_table is int32 [sequences, entries], got {page_table.dtype} {tuple(page_table.shape)}")
    if page_table.get_device() != device.index:
        raise ValueError(f"{what}: all tensors must be on {device}, got page_table on {page_table.device}")
    sequences, entries = page_table.shape
    pitch = entries
    if not page_table.is_contiguous():
        if (entries > 1 and page_table.stride(1) != 1) or (sequences > 1 and page_table.stride(0) < entries):
            page_table = page_table.contiguous()
        elif sequences > 1:
            pitch = page_table.stride(0)
    keys, values = cache
    pages, page_size, branches, routing_dim = keys.shape
    width, value_dim = branches * routing_dim, values.shape[2]
    key_page, value_page = page_size * width, page_size * value_dim
    if pages > 1:
        key_page, value_page = keys.stride(0), values.stride(0)
    args = _lib.PagedCacheArgs(
        keys.data_ptr(), key_page, values.data_ptr(), value_page, pages, page_size, width, value_dim, page_table.data_ptr(), pitch,
        entries,
    )
    return args, page_table


def _rows16(t: Tensor, width: int) -> tuple[Tensor, int]:
    """``[N, ...]`` rows as 16-byte aligned ones of ``width`` elements, and their pitch."""

    if t.is_contiguous() and not t.data_ptr() % 16:   # the usual case; 1.4 us of the host's time less
        return t, width
    t = t.detach().reshape(t.shape[0], width)
    pitch = t.stride(0) if t.shape[0] > 1 else width
    if t.stride(1) != 1 or pitch < width or pitch % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        pitch = width
    return t, pitch


def cache_append_hip(
    cache: PagedCache, key: Tensor, value: Tensor, page_table: Tensor, lengths: Tensor, offsets: Tensor,
    *, max_chunk: int | None = None,
) -> None:
    """Writes new tokens into their pages.

    ``key`` ``[N, branches, R]`` and ``value`` ``[N, D]`` of the cache's types
    are the new tokens of all sequences, packed: those of sequence b are rows
    ``offsets[b]`` to ``offsets[b + 1]`` (int32 ``[sequences + 1]``) and become
    its last ones, ``lengths`` (int32 ``[sequences]``) being the lengths with
    them.  Rows in front of ``offsets[0]`` and behind ``offsets[-1]`` belong to
    no sequence.  Tokens whose page the table does not name (an entry outside
    of the cache, a position behind its entries) are dropped.  ``max_chunk``:
    the largest number of new tokens of a sequence, where the program knows it
    (it chooses the launch, not the result).
    """

    what = "cache_append_hip"
    _no_grad(what, key, value, *cache)
    device = _check_cache(what, cache)
    keys, values = cache
    if key.dtype is not keys.dtype or key.shape[1:] != keys.shape[2:] or key.ndim != 3:
        raise ValueError(f"{what}: key is {keys.dtype} [N, {keys.shape[2]}, {keys.shape[3]}], got {key.dtype} {tuple(key.shape)}")
    if value.dtype is not values.dtype or value.shape != (key.shape[0], values.shape[2]):
        raise ValueError(f"{what}: value is {values.dtype} [{key.shape[0]}, {values.shape[2]}], got {value.dtype} {tuple(value.shape)}")
    for t in (key, value):
        if t.get_device() != device.index:
            raise ValueError(f"{what}: all tensors must be on {device}, got one on {t.device}")
    args, page_table = _cache_args(what, cache, page_table, device)
    sequences = page_table.shape[0]
    lengths = _check_int32(what, "lengths", lengths, (sequences,), device)
    offsets = _check_int32(what, "offsets", offsets, (sequences + 1,), device)
    key, ldk = _rows16(key, args.key_width)
    value, ldv = _rows16(value, args.value_dim)
    _launch(what, device, _lib.get().da_cache_append, ctypes.byref(args), key.data_ptr(), ldk, value.data_ptr(), ldv, key.shape[0],
            lengths.data_ptr(), offsets.data_ptr(), sequences, _hint(what, "max_chunk", max_chunk))


def _hint(what: str, name: str, value: int | None) -> int:
    if value is None:
        return 0
    if value < 1:
        raise ValueError(f"{what}: {name} is at least 1")
    return int(value)


def _paged_attention(what, query, cache, page_table, lengths, offsets, scales, weights, want_weights, mix, causal, max_chunk,
                     max_length, weights_out):
    _no_grad(what, query, scales, mix, weights, *cache)
    device = _check_cache(what, cache)
    keys, values = cache
    _, page_size, branches, routing_dim = keys.shape
    if query.dtype is not keys.dtype or query.ndim != 3 or query.shape[1:] != keys.shape[2:]:
        raise ValueError(f"{what}: query is {keys.dtype} [N, {branches}, {routing_dim}], got {query.dtype} {tuple(query.shape)}")
    scales_code = _CODES.get(scales.dtype)
    if scales_code is None or scales.ndim != 1 or scales.shape[0] < 1:
        raise ValueError(f"{what}: scales are a floating vector, one for each map, got {scales.dtype} {tuple(scales.shape)}")
    maps = scales.shape[0]
    if maps > MAX_MAPS or max(maps, branches) % min(maps, branches):
        raise NotImplementedError(f"{what}: {maps} maps of {branches} branches (multiples of each other, at most {MAX_MAPS} maps)")
    score_dim, _, repeat, mult = routed_score_layout(branches, maps, routing_dim)
    if score_dim % 64 or score_dim > 512:
        raise NotImplementedError(f"{what}: score widths are multiples of 64 up to 512, not {score_dim}")
    for name, t in (("query", query), ("scales", scales), ("mix", mix), ("weights", weights), ("out", weights_out)):
        if t is not None and t.get_device() != device.index:
            raise ValueError(f"{what}: all tensors must be on {device}, got {name} on {t.device}")
    if mix is not None and (mix.dtype is not _FLOAT32 or mix.shape != (maps,)):
        raise ValueError(f"{what}: mix is float32 of shape ({maps},), got {mix.dtype} {tuple(mix.shape)}")
    cache_args, page_table = _cache_args(what, cache, page_table, device)
    sequences, entries = page_table.shape
    lengths = _check_int32(what, "lengths", lengths, (sequences,), device)
    offsets = _check_int32(what, "offsets", offsets, (sequences + 1,), device)
    rows = query.shape[0]
    query, ldq = _rows16(query, branches * routing_dim)
    scales = scales.detach().contiguous()
    if mix is not None:
        mix = mix.detach().contiguous()
    shape = (rows, values.shape[2]) if mix is not None else (rows, maps, values.shape[2])
    out = torch.empty(shape, dtype=values.dtype, device=device)
    weights_shape = (sequences, entries * page_size)
    for name, t in (("weights", weights), ("out", weights_out)):
        if t is not None and (t.dtype is not _FLOAT32 or t.shape != weights_shape):
            raise ValueError(f"{what}: {name} is float32 of shape {weights_shape}, got {t.dtype} {tuple(t.shape)}")
    if weights_out is not None and not weights_out.is_contiguous():
        raise ValueError(f"{what}: out is contiguous")
    if want_weights:
        if weights is not None:
            weights = weights.detach().contiguous()
        if weights_out is None:
            weights_out = torch.empty(weights_shape, dtype=_FLOAT32, device=device)
    if sequences == 0:
        if rows:
            raise ValueError(f"{what}: rows without sequences")
        return out, weights_out
    args = _lib.PagedAttentionArgs(
        cache_args, query.data_ptr(), ldq, rows, lengths.data_ptr(), offsets.data_ptr(), sequences, scales.data_ptr(), scales_code,
        mult, maps, score_dim, repeat, int(causal), None if mix is None else mix.data_ptr(), _HALF_CODES[keys.dtype],
        _HALF_CODES[values.dtype], out.data_ptr(), None if weights is None else weights.data_ptr(),
        None if weights_out is None else weights_out.data_ptr(), weights_shape[1], _hint(what, "max_chunk", max_chunk),
        _hint(what, "max_length", max_length),
    )
    lib = _lib.get()
    args_p = ctypes.byref(args)
    nbytes = lib.da_paged_attention_workspace_bytes(args_p)
    if nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
    _launch(what, device, lib.da_paged_attention, args_p)
    return out, weights_out


def paged_attention_hip(
    query: Tensor, cache: PagedCache, page_table: Tensor, lengths: Tensor, offsets: Tensor, scales: Tensor, causal: bool = True,
    *, mix: Tensor | None = None, max_chunk: int | None = None, max_length: int | None = None,
) -> Tensor:
    """The outer attention of new tokens over their sequences' cached tokens.

    ``query`` ``[N, branches, R]``: the routed query rows of the new tokens,
    packed as for ``cache_append_hip``, which has put their keys and values into
    the cache.  Maps (one for each of ``scales``, fp32 or 16-bit) are assembled
    from the branches as by ``assemble_score_maps``.  A new token sees the
    tokens up to its own (``causal``), or all of its sequence.  Returns ``[N,
    maps, D]`` of the values' type, or with ``mix`` (fp32 ``[maps]``) the maps'
    sum with these weights, ``[N, D]``.  Rows of no sequence, and rows that see
    nothing, are zero.  Scores, softmax and sums are fp32; probabilities are
    rounded to the values' type for their product, the result once.  An
    infinity or a NaN in a value reaches the rows that see its token, one in a
    key the maps that read it, too.
    ``max_chunk`` and ``max_length``: the largest numbers of new and of all
    tokens of a sequence, where the program knows them (they choose the launch,
    not the result; without the first a call is launched as if all rows were one
    sequence's, and single tokens of 64 sequences take 73 us instead of 40).
    """

    return _paged_attention("paged_attention_hip", query, cache, page_table, lengths, offsets, scales, None, False, mix, causal,
                            max_chunk, max_length, None)[0]


def paged_attention_weights_hip(
    query: Tensor, cache: PagedCache, page_table: Tensor, lengths: Tensor, offsets: Tensor, scales: Tensor, causal: bool = True,
    *, weights: Tensor | None = None, out: Tensor | None = None, mix: Tensor | None = None, max_chunk: int | None = None,
    max_length: int | None = None,
) -> tuple[Tensor, Tensor]:
    """``paged_attention_hip`` and the weights that the cached tokens gathered.

    Returns ``(attention, gathered)``: ``gathered`` fp32 ``[sequences, entries *
    page_size]`` is ``weights`` (None: zeros) plus, for each cached token, the
    probabilities that this call's rows and maps gave it.  Tokens that are new
    in this call start from zero whatever ``weights`` has there; behind a
    sequence's last token it is zero.  ``out`` takes the result and may be
    ``weights`` itself.
    """

    return _paged_attention("paged_attention_weights_hip", query, cache, page_table, lengths, offsets, scales, weights, True, mix,
                            causal, max_chunk, max_length, out)


def cache_select_hip(weights: Tensor, lengths: Tensor, keep: int, recent: int = 0) -> tuple[Tensor, Tensor]:
    """The tokens that stay when sequences are cut to ``keep`` tokens each.

    Of sequence b (``lengths[b]`` tokens with the ``weights`` fp32 ``[sequences,
    capacity]``) the last ``recent`` stay, and of the others those of the
    largest weights, equal ones in their order (a NaN is below everything).
    Returns ``(kept, counts)``: int32 ``[sequences, keep]``, ascending, -1 behind
    the ``counts[b]`` that stay (all of a sequence that is not longer).
    """

    what = "cache_select_hip"
    _no_grad(what, weights)
    if weights.dtype is not _FLOAT32 or weights.ndim != 2:
        raise ValueError(f"{what}: weights are float32 [sequences, capacity], got {weights.dtype} {tuple(weights.shape)}")
    if not weights.is_cuda:
        raise ValueError(f"{what}: HIP kernels require tensors on a ROCm device")
    if not 0 <= recent <= keep:
        raise ValueError(f"{what}: needs 0 <= recent <= keep, got {recent} and {keep}")
    device = weights.device
    sequences, capacity = weights.shape
    lengths = _check_int32(what, "lengths", lengths, (sequences,), device)
    weights = weights.detach()
    if (capacity > 1 and weights.stride(1) != 1) or (sequences > 1 and weights.stride(0) < capacity):
        weights = weights.contiguous()
    kept = torch.empty(sequences, keep, dtype=_INT32, device=device)
    counts = torch.empty(sequences, dtype=_INT32, device=device)
    _launch(what, device, _lib.get().da_cache_select, weights.data_ptr(), weights.stride(0) if sequences > 1 else capacity, capacity,
            lengths.data_ptr(), sequences, keep, recent, kept.data_ptr(), counts.data_ptr())
    return kept, counts


def cache_compact_hip(
    cache: PagedCache, page_table: Tensor, kept: Tensor, counts: Tensor, out_cache: PagedCache, out_page_table: Tensor,
    *, weights: Tensor | None = None,
) -> Tensor | None:
    """Moves the kept tokens into other pages, in order.

    Token ``kept[b, i]`` of sequence b becomes token i, for ``i < counts[b]``
    (``cache_select_hip``).  ``out_cache`` may be the cache itself: the pages that
    ``out_page_table`` names must then be other ones than those that kept tokens
    come from.  Returns the ``weights`` (fp32 ``[sequences, capacity]``) of the
    moved tokens at their new places, zero behind them, or None.
    """

    what = "cache_compact_hip"
    _no_grad(what, weights, *cache, *out_cache)
    device = _check_cache(what, cache)
    if _check_cache(what, out_cache) != device:
        raise ValueError(f"{what}: all tensors must be on {device}, got one on {out_cache.keys.device}")
    if (cache.keys.dtype, cache.values.dtype) != (out_cache.keys.dtype, out_cache.values.dtype) or (
        cache.keys.shape[2:] != out_cache.keys.shape[2:] or cache.values.shape[2] != out_cache.values.shape[2]
    ):
        raise ValueError(f"{what}: the caches' types and widths must match")
    source, page_table = _cache_args(what, cache, page_table, device)
    target, out_page_table = _cache_args(what, out_cache, out_page_table, device)
    sequences = page_table.shape[0]
    if out_page_table.shape[0] != sequences or kept.ndim != 2:
        raise ValueError(f"{what}: kept and both page tables have a row for each sequence")
    kept = _check_int32(what, "kept", kept, (sequences, kept.shape[1]), device)
    counts = _check_int32(what, "counts", counts, (sequences,), device)
    moved = None
    if weights is not None:
        shape = (sequences, page_table.shape[1] * cache.page_size)
        if weights.dtype is not _FLOAT32 or weights.shape != shape:
            raise ValueError(f"{what}: weights are float32 of shape {shape}, got {weights.dtype} {tuple(weights.shape)}")
        if weights.get_device() != device.index:
            raise ValueError(f"{what}: all tensors must be on {device}, got weights on {weights.device}")
        weights = weights.detach().contiguous()
        moved = torch.empty(sequences, out_page_table.shape[1] * out_cache.page_size, dtype=_FLOAT32, device=device)
    if sequences == 0:
        return moved
    _launch(what, device, _lib.get().da_cache_compact, ctypes.byref(source), ctypes.byref(target), sequences, kept.data_ptr(),
            kept.shape[1], kept.shape[1], counts.data_ptr(), None if weights is None else weights.data_ptr(),
            0 if weights is None else weights.shape[1], None if moved is None else moved.data_ptr(),
            0 if moved is None else moved.shape[1])
    return moved


class TokenLogProbs(NamedTuple):
    """What ``token_log_probs_hip`` returns; all fp32 but the tokens (int64)."""

    log_probs: Tensor                  # [...]: of the given tokens
    entropy: Tensor | None             # [...]
    top_log_probs: Tensor | None       # [..., top]
    top_tokens: Tensor | None          # [..., top]


def _logit_rows(logits: Tensor) -> tuple[Tensor, int]:
    """The logits as rows with unit column stride, and their pitch."""

    vocab = logits.shape[-1]
    rows = logits.detach()
    rows = rows if rows.ndim == 2 else rows.reshape(-1, vocab)
    if (vocab > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < vocab):
        rows = rows.contiguous()
    return rows, rows.stride(0) if rows.shape[0] > 1 else vocab


def _token_log_probs(logits: Tensor, tokens: Tensor, top: int, entropy: bool, ignore_index: int, want_lse: bool):
    what = "token_log_probs_hip"
    lead, device = logits.shape[:-1], logits.device
    rows, pitch = _logit_rows(logits)
    tokens = tokens.contiguous()
    count, vocab = rows.shape

    def new(*shape: int, dtype: torch.dtype = _FLOAT32) -> Tensor:
        return torch.empty(*lead, *shape, dtype=dtype, device=device)

    log_probs = new()
    entropies = new() if entropy else None
    lse = new(2) if want_lse else None
    top_log_probs, top_tokens = (new(top), new(top, dtype=_INT64)) if top else (None, None)
    lib = _lib.get()
    nbytes = lib.da_token_log_probs_workspace_bytes(count, vocab, top)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _launch(what, device, lib.da_token_log_probs, rows.data_ptr(), count, vocab, pitch, _CODES[logits.dtype], tokens.data_ptr(),
            ignore_index, log_probs.data_ptr(), None if entropies is None else entropies.data_ptr(),
            None if lse is None else lse.data_ptr(), top, None if not top else top_log_probs.data_ptr(),
            None if not top else top_tokens.data_ptr(), None if workspace is None else workspace.data_ptr(), nbytes)
    return log_probs, entropies, top_log_probs, top_tokens, lse


class _TokenLogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, entropy, ignore_index):  # type: ignore[override]
        log_probs, entropies, top_log_probs, top_tokens, lse = _token_log_probs(logits, tokens, top, entropy, ignore_index, True)
        ctx.save_for_backward(logits, tokens, lse, entropies, top_tokens)
        ctx.top, ctx.ignore_index = top, ignore_index
        ctx.set_materialize_grads(False)
        if top_tokens is not None:
            ctx.mark_non_differentiable(top_tokens)
        return log_probs, entropies, top_log_probs, top_tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_log_probs, g_entropy=None, g_top=None, _=None):  # type: ignore[override]
        logits, tokens, lse, entropies, top_tokens = ctx.saved_tensors
        if (g_log_probs is None and g_entropy is None and g_top is None) or not ctx.needs_input_grad[0]:
            return None, None, None, None, None
        what = "token_log_probs_hip backward"
        rows, pitch = _logit_rows(logits)
        tokens = tokens.contiguous()
        g_log_probs, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_log_probs, g_entropy, g_top))
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _launch(what, logits.device, _lib.get().da_token_log_probs_backward, rows.data_ptr(), rows.shape[0], rows.shape[1], pitch,
                _CODES[logits.dtype], tokens.data_ptr(), ctx.ignore_index, lse.data_ptr(),
                None if entropies is None else entropies.data_ptr(), ctx.top, None if top_tokens is None else top_tokens.data_ptr(),
                *(None if g is None else g.data_ptr() for g in (g_log_probs, g_entropy, g_top)), grad.data_ptr(), rows.shape[1])
        return grad, None, None, None, None


def token_log_probs_hip(
    logits: Tensor, tokens: Tensor, *, top: int = 0, entropy: bool = True, ignore_index: int = -100
) -> TokenLogProbs:
    """Log probabilities of ``tokens`` (int64 ``[...]``) under ``logits`` ``[...,
    vocab]`` (fp32, fp16 or bf16), the distributions' entropies (in nats; None
    unless wanted), and the ``top`` (at most 64) most probable tokens with their
    log probabilities, equal logits in the order of their tokens.

    A token that is ``ignore_index`` has the log probability 0 and no gradient;
    one outside the vocabulary has NaN (its row's gradient, too).  Rows with a
    NaN or +infinity, and rows of -infinity throughout, have NaN log
    probabilities, as ``log_softmax``.  Statistics are fp32.  Differentiable in
    the logits through all three (in reverse mode); the gradient is rounded once
    to their type.
    """

    what = "token_log_probs_hip"
    if logits.dtype not in _CODES:
        raise ValueError(f"{what}: logits are float32, float16 or bfloat16, got {logits.dtype}")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits are [..., vocab], got shape {tuple(logits.shape)}")
    if tokens.dtype is not _INT64 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: tokens are int64 of shape {tuple(logits.shape[:-1])}, got {tokens.dtype} {tuple(tokens.shape)}")
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise NotImplementedError(f"{what}: top is at most {MAX_TOP} and the vocabulary, got {top}")
    if not logits.is_cuda:
        raise ValueError(f"{what}: HIP kernels require tensors on a ROCm device")
    if tokens.get_device() != logits.get_device():
        raise ValueError(f"{what}: all tensors must be on {logits.device}, got tokens on {tokens.device}")
    if forward_ad._current_level >= 0 and _has_tangent(logits):
        raise ValueError(f"{what} has no forward-mode derivative: detach its inputs")
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogProbs(*_TokenLogProbsFunction.apply(logits, tokens, top, entropy, ignore_index))
    return TokenLogProbs(*_token_log_probs(logits, tokens, top, entropy, ignore_index, False)[:4])


__all__ = [
    "PagedCache",
    "TokenLogProbs",
    "cache_append_hip",
    "cache_compact_hip",
    "cache_select_hip",
    "paged_attention_hip",
    "paged_attention_weights_hip",
    "paged_cache",
    "token_log_probs_hip",
]
