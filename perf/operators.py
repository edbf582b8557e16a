"""Performance cases of the framework's 8-bit operators.

Three operators that share one 8-bit format (signed integers from -127 to 127
with an fp32 scale for each row, or for each 128 columns of a row):

* the linear layer on 8-bit integers, a scale for each token and one for each
  output channel, with bias, GELU and residual;
* the root-mean-square norm with the residual's addition in front of it, its
  output in 8 bits for that linear layer or in 16 bits with a backward pass;
* activation checkpoints in 8 bits: rows kept and restored, and GELU with its
  backward pass from the kept rows.

``listed()`` holds the cases that are reported, ``draw()`` more of the same
ranges, ``run()`` one pass (in plain 32-bit torch, or with ``own`` through the
framework), ``exact()`` the same results in 64 bits.  Rows kept in 8 bits come
back as the values they stand for, in the 16-bit type they were made from.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_GROUP = 128
_EPS = 1e-6
# The smallest scale: an all-zero row has this one, and its values are zero.
_LEAST_SCALE = 2.0 ** -126


def _linear(name: str, rows: int, inner: int, outer: int, **options) -> dict:
    case = {"kind": "linear", "rows": rows, "inner": inner, "outer": outer, "dtype": "bf16", "quantized": False,
            "bias": True, "gelu": False, "residual": False, **options}
    return {"name": name, **case} if name else case


def _norm(name: str, kind: str, rows: int, width: int, **options) -> dict:
    case = {"kind": kind, "rows": rows, "width": width, "dtype": "bf16", "residual": True, **options}
    return {"name": name, **case} if name else case


def _saved(name: str, kind: str, rows: int, width: int, **options) -> dict:
    case = {"kind": kind, "rows": rows, "width": width, "dtype": "bf16", **options}
    return {"name": name, **case} if name else case


def listed() -> list[dict]:
    return [
        # The feed-forward's first linear for one new token: latency counts.
        _linear("linear-token", 1, 512, 1536, gelu=True),
        # A few sequences' tokens against a wide layer: the weights' bytes.
        _linear("linear-few", 16, 4096, 4096, residual=True),
        # The feed-forward's first linear over the language model's batch.
        _linear("linear-ffn", 4096, 512, 1536, gelu=True),
        # Odd sizes everywhere, fp16, the second linear's residual.
        _linear("linear-ragged", 777, 1000, 1111, dtype="fp16", residual=True),
        # A wide layer over a long prompt, rows already in 8 bits (a norm's output).
        _linear("linear-wide", 8192, 4096, 4096, quantized=True, bias=False),
        # The norm in front of the feed-forward, one token.
        _norm("norm-token", "norm", 1, 512),
        # The same over the language model's batch, the sum already formed.
        _norm("norm-lm", "norm", 4096, 512, residual=False),
        # A training step of the norm at an odd width, fp16.
        _norm("norm-train", "norm-train", 3885, 1001, dtype="fp16"),
        # A wide model's norm over a long prompt.
        _norm("norm-wide", "norm", 16384, 4096),
        # A linear layer's input kept for the backward pass, odd sizes.
        _saved("save-ragged", "save", 3885, 1111, dtype="fp16"),
        # GELU of the feed-forward, forward and backward from the kept rows.
        _saved("gelu-lm", "gelu", 4096, 1536),
        # The same for a wide model's long batch.
        _saved("gelu-wide", "gelu", 16384, 6144),
    ]


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    """One more case: sizes spread over their logarithm, mostly odd ones for
    the widths, both 16-bit types."""

    kind = rng.choice(("linear", "linear", "linear", "norm", "norm", "norm-train", "save", "gelu", "gelu"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    rows = _log_int(rng, 1, 16384)

    def width(high: int) -> int:
        # Model widths are multiples of 64; the others are what a user may have.
        n = _log_int(rng, 64, high)
        return n // 64 * 64 if rng.random() < 0.6 else n

    if kind == "linear":
        inner, outer = width(4096), width(6144)
        rows = max(1, min(rows, 8192 * 4096 * 4096 // (inner * outer)))
        return _linear("", rows, inner, outer, dtype=dtype, quantized=rng.random() < 0.3, bias=rng.random() < 0.6,
                       gelu=rng.random() < 0.4, residual=rng.random() < 0.4)
    if kind in ("norm", "norm-train"):
        return _norm("", kind, rows, width(4096), dtype=dtype, residual=rng.random() < 0.7)
    return _saved("", kind, rows, width(6144), dtype=dtype)


def _rows(rows: int, width: int, spread: float = 1.0):
    """Activations of a residual stream: normal, with a few channels that are
    several times larger, as trained models have them."""

    gain = torch.where(torch.rand(width) < 0.01, 8.0, 1.0) * (0.5 + torch.rand(width))
    return torch.randn(rows, width) * gain * spread


def _padded_rows(values):
    """8-bit rows at a pitch of a multiple of 16 bytes, as a program keeps
    them; the columns behind a row are not part of it."""

    rows, width = values.shape
    store = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.int8)
    store[:, :width] = values
    return store[:, :width]


def prepare(case: dict, seed: int) -> dict:
    dtype = _DTYPES[case["dtype"]]
    torch.manual_seed(seed)
    state = {"case": case, "dtype": dtype}
    with torch.device("cuda"):
        if case["kind"] == "linear":
            rows, inner, outer = case["rows"], case["inner"], case["outer"]
            weight = torch.randn(outer, inner) * inner ** -0.5 * (0.5 + torch.rand(outer, 1))
            scales = weight.abs().amax(1, keepdim=True) / 127
            state["weight"] = _padded_rows(torch.round(weight / scales).to(torch.int8))
            state["weight_scales"] = scales
            x = _rows(rows, inner)
            if case["quantized"]:
                scales = x.abs().amax(1, keepdim=True) / 127
                state["x"] = _padded_rows(torch.round(x / scales).to(torch.int8))
                state["x_scales"] = scales
            else:
                state["x"] = x.to(dtype)
            state["bias"] = (0.1 * torch.randn(outer)).to(dtype) if case["bias"] else None
            state["residual"] = _rows(rows, outer).to(dtype) if case["residual"] else None
            return state
        rows, width = case["rows"], case["width"]
        state["x"] = _rows(rows, width).to(dtype)
        if case["kind"] in ("norm", "norm-train"):
            state["residual"] = _rows(rows, width, 2.0).to(dtype) if case["residual"] else None
            state["weight"] = (1 + 0.2 * torch.randn(width)).to(dtype)
        if case["kind"] in ("norm-train", "gelu"):
            state["grad"] = torch.randn(rows, width).to(dtype)
        if case["kind"] == "norm-train":
            # The gradient that reaches the sum past the norm.
            state["grad_sum"] = torch.randn(rows, width).to(dtype)
    return state


# ---- plain forms, 32 bits ---------------------------------------------------


def _kept(x):
    """``(values, scale)`` of 32-bit rows in 8 bits, one scale a row."""

    scale = (x.abs().amax(-1, keepdim=True) * (1 / 127)).clamp_min(_LEAST_SCALE)
    return torch.clamp(torch.round(x / scale), -127, 127), scale


def _kept_groups(x):
    """The values that 32-bit rows kept in groups of 128 columns stand for."""

    rows, width = x.shape
    groups = -(-width // _GROUP)
    padded = x.new_zeros(rows, groups * _GROUP)
    padded[:, :width] = x
    values, scale = _kept(padded.view(rows, groups, _GROUP))
    return (values * scale).view(rows, -1)[:, :width]


def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))


def _plain(state: dict):
    case, dtype = state["case"], state["dtype"]
    kind = case["kind"]
    if kind == "linear":
        if case["quantized"]:
            values, scale = state["x"].float(), state["x_scales"]
        else:
            values, scale = _kept(state["x"].float())
        y = values @ state["weight"].float().t() * scale * state["weight_scales"].view(1, -1)
        if state["bias"] is not None:
            y = y + state["bias"].float()
        if case["gelu"]:
            y = _gelu(y)
        y = y.to(dtype)
        return y if state["residual"] is None else (y.float() + state["residual"].float()).to(dtype)
    if kind in ("norm", "norm-train"):
        total = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(dtype)
        s, w = total.float(), state["weight"].float()
        factor = torch.rsqrt((s * s).mean(-1, keepdim=True) + _EPS)
        unit = s * factor
        if kind == "norm":
            values, scale = _kept(unit * w)
            return {"normalized": (values * scale).to(dtype), "sum": total}
        g = state["grad"].float()
        gw = g * w
        grad_x = factor * (gw - unit * (gw * unit).mean(-1, keepdim=True)) + state["grad_sum"].float()
        return {"normalized": (unit * w).to(dtype), "sum": total, "grad_x": grad_x.to(dtype),
                "grad_weight": (g * unit).sum(0).to(dtype)}
    if kind == "save":
        return _kept_groups(state["x"].float()).to(dtype)
    z = state["x"].float()
    kept = _kept_groups(z)
    below = 0.5 * (1 + torch.erf(kept * 0.5 ** 0.5))
    slope = below + kept * torch.exp(-0.5 * kept * kept) * (2 * math.pi) ** -0.5
    # Forward: GELU of z.  Backward, from the kept rows: the gradient at z,
    # and GELU again for the weight gradient of the layer behind it.
    return {"out": _gelu(z).to(dtype), "grad": (state["grad"].float() * slope).to(dtype), "again": (kept * below).to(dtype)}


# ---- the framework's calls --------------------------------------------------


def _package():
    at = os.path.join(_ROOT, "double-attention_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import double_attention

    return double_attention


def _own(state: dict):
    da = _package()
    case, dtype = state["case"], state["dtype"]
    kind = case["kind"]
    if kind == "linear":
        x = da.QuantizedRows(state["x"], state["x_scales"]) if case["quantized"] else state["x"]
        weight = da.QuantizedRows(state["weight"], state["weight_scales"])
        return da.linear_int8_hip(x, weight, state["bias"], activation="gelu" if case["gelu"] else None,
                                  residual=state["residual"], dtype=dtype)
    if kind == "norm":
        kept, total = da.add_rms_norm_int8_hip(state["x"], state["residual"], state["weight"], _EPS)
        return {"normalized": da.dequantize_int8_hip(kept, dtype), "sum": total}
    if kind == "norm-train":
        normalized, total = da.add_rms_norm_hip(state["x"], state["residual"], state["weight"], _EPS)
        grad_x, grad_weight = da.add_rms_norm_backward_hip(total, state["grad"], state["grad_sum"], state["weight"], _EPS)
        return {"normalized": normalized, "sum": total, "grad_x": grad_x, "grad_weight": grad_weight}
    if kind == "save":
        return da.dequantize_int8_hip(da.quantize_int8_hip(state["x"], da.INT8_GROUP), dtype)
    out, kept = da.gelu_int8_hip(state["x"])
    grad, again = da.gelu_int8_backward_hip(kept, state["grad"])
    return {"out": out, "grad": grad, "again": again}


def run(state: dict):
    return _own(state) if own else _plain(state)


def work(case: dict) -> dict:
    rows, kind = case["rows"], case["kind"]
    if kind == "linear":
        inner, outer = case["inner"], case["outer"]
        inputs = rows * (inner + 4) if case["quantized"] else 2 * rows * inner
        outputs = 2 * rows * outer * (2 if case["residual"] else 1)
        return {"bytes": inputs + outer * (inner + 4) + outputs + (2 * outer if case["bias"] else 0),
                "flops": 2 * rows * inner * outer}
    cells, width = rows * case["width"], case["width"]
    if kind == "norm":
        # x and the residual read, the sum and the normalized rows written
        # (without a residual the sum is x itself).
        return {"bytes": 2 * cells * (4 if case["residual"] else 2) + 2 * width, "flops": 8 * cells}
    if kind == "norm-train":
        # Forward, then the sum and two gradients read and one written.
        return {"bytes": 2 * cells * ((4 if case["residual"] else 2) + 4) + 6 * width, "flops": 18 * cells}
    if kind == "save":
        # Read; kept in a byte, read again; written.
        return {"bytes": 6 * cells + 8 * rows * -(-width // _GROUP), "flops": 6 * cells}
    # Forward: z read, GELU and the kept byte written.  Backward: the byte and
    # the gradient read, the gradient at z and GELU written.
    return {"bytes": (2 + 2 + 1 + 1 + 2 + 2 + 2) * cells + 8 * rows * -(-width // _GROUP), "flops": 60 * cells}


# ---- the same results in 64 bits --------------------------------------------


def _stands_for(x, width: int):
    """What rows of 64-bit numbers stand for once kept in 8 bits, a scale for
    every ``width`` columns."""

    parts = []
    for part in x.split(width, dim=-1):
        largest = part.abs().max(dim=-1, keepdim=True).values
        steps = torch.where(largest > 0, largest / 127, torch.ones_like(largest))
        parts.append(torch.floor(part / steps + 0.5).clamp(-127, 127) * steps)
    return torch.cat(parts, dim=-1)


def _normal_cdf(x):
    return torch.special.ndtr(x)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind, dtype = case["kind"], state["dtype"]
    x = state["x"].double()
    if kind == "linear":
        rows = x * state["x_scales"].double() if case["quantized"] else _stands_for(x, case["inner"])
        weight = state["weight"].double() * state["weight_scales"].double()
        y = torch.mm(rows, weight.t())
        if case["bias"]:
            y += state["bias"].double()
        if case["gelu"]:
            y = y * _normal_cdf(y)
        return y + state["residual"].double() if case["residual"] else y
    if kind in ("norm", "norm-train"):
        # The sum is a 16-bit tensor that the model carries on; the norm is of it.
        s = x if state["residual"] is None else (x + state["residual"].double()).to(dtype).double()
        w = state["weight"].double()
        length = (s.square().sum(-1, keepdim=True) / case["width"] + _EPS).sqrt()
        if kind == "norm":
            return {"normalized": _stands_for(s / length * w, case["width"]), "sum": s}
        s.requires_grad_(True)
        w.requires_grad_(True)
        y = s / (s.square().sum(-1, keepdim=True) / case["width"] + _EPS).sqrt() * w
        both = (y * state["grad"].double()).sum() + (s * state["grad_sum"].double()).sum()
        grad_x, grad_weight = torch.autograd.grad(both, (s, w))
        return {"normalized": y.detach(), "sum": s.detach(), "grad_x": grad_x, "grad_weight": grad_weight}
    if kind == "save":
        return _stands_for(x, _GROUP)
    kept = _stands_for(x, _GROUP).requires_grad_(True)
    again = kept * _normal_cdf(kept)
    (grad,) = torch.autograd.grad(again, kept, state["grad"].double())
    return {"out": x * _normal_cdf(x), "grad": grad, "again": again.detach()}
