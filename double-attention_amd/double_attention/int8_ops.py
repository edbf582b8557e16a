"""8-bit operators of the blocks' feed-forward on the gfx950 kernels.

Three operators around one format (``QuantizedRows``: signed integers from
-127 to 127 with an fp32 scale for each row, or for each 128 columns of it):

* ``linear_int8_hip``: the linear layer on 8-bit integers, one scale per token
  and per output channel, with bias, GELU and residual;
* ``add_rms_norm_int8_hip`` and ``add_rms_norm_hip``: the root-mean-square
  norm with the residual's addition in front of it, for that linear layer in
  8 bits, or in 16 bits with a backward pass;
* ``gelu_int8_hip`` / ``gelu_int8_backward_hip``, and ``quantize_int8_hip`` /
  ``dequantize_int8_hip`` in groups of 128: activations that the backward pass
  finds in 8 bits.

As in ``hip_ops``, PyTorch supplies memory and the current stream, and nothing
falls back to another implementation: a call the kernels do not cover raises.
``add_rms_norm_hip`` is differentiable; the other calls refuse tensors whose
gradients autograd would record.
The kernels run on the inputs' device, whichever is current.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from .hip_ops import _stream, dtype_code

INT8_GROUP = _lib.INT8_GROUP
# Columns of rows with one scale each, and widths of the norm.
MAX_ROW_COLUMNS = 65536
MAX_NORM_WIDTH = 16384


class QuantizedRows(NamedTuple):
    """Rows in 8 bits.

    ``values`` is int8 ``[..., columns]``, ``scales`` fp32 ``[..., G]``: G = 1
    (``group`` None, a scale for each row) or the columns' groups of 128
    (``group`` 128).  ``values * scale`` is what the rows stand for.  A row
    (group) whose scale is NaN held an infinity or a NaN.  ``values`` made
    here are views of rows padded to a multiple of 16 bytes, the pitch the
    kernels read; others are copied into such rows in each call.
    """

    values: Tensor
    scales: Tensor
    group: int | None = None


# The private call skips torch.cuda's own checks; a torch without device support has none.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_INT8, _FLOAT32 = torch.int8, torch.float32
_CODES = {torch.float32: _lib.DA_F32, torch.float16: _lib.DA_F16, torch.bfloat16: _lib.DA_BF16}
_HALF_CODES = {torch.float16: _lib.DA_F16, torch.bfloat16: _lib.DA_BF16}


def _launch(what: str, device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` on ``device``, which need not be the current one."""

    if device.index == _current_device():
        rc = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device))
    if rc:
        _lib.check(rc, what)


def _check_input(what: str, x: Tensor, codes: dict = _HALF_CODES) -> int:
    """The dtype code of ``x``: rows of at least one column on a device."""

    code = codes.get(x.dtype)
    if code is None:
        names = " or ".join(str(t).removeprefix("torch.") for t in codes)
        raise ValueError(f"{what}: HIP kernels require {names} tensors, got {x.dtype}")
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: expected rows of at least one column, got shape {tuple(shape)}")
    if not x.is_cuda:
        raise ValueError(f"{what}: HIP kernels require tensors on a ROCm device")
    return code


def _check_on(what: str, device: torch.device, t: Tensor) -> None:
    if t.get_device() != device.index:
        raise ValueError(f"{what}: all tensors must be on {device}, got one on {t.device}")


def _check_like(what: str, x: Tensor, t: Tensor) -> None:
    if t.shape != x.shape or t.dtype is not x.dtype:
        raise ValueError(f"{what}: expected shape {tuple(x.shape)} and {x.dtype}, got {tuple(t.shape)} and {t.dtype}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{what}: all tensors must be on {x.device}, got one on {t.device}")


def _check_param(what: str, device: torch.device, t: Tensor, size: int) -> int:
    code = _CODES.get(t.dtype)
    if code is None or t.shape != (size,):
        raise ValueError(f"{what}: expected a floating parameter of shape ({size},), got {t.dtype} {tuple(t.shape)}")
    _check_on(what, device, t)
    return code


def _has_tangent(*tensors: Tensor | None) -> bool:
    """Whether one of the tensors carries a forward-mode tangent (under
    torch.no_grad(), too).  There are tangents from level 0 on."""

    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _no_grad(what: str, *tensors: Tensor | None) -> None:
    if forward_ad._current_level >= 0 and _has_tangent(*tensors):
        raise ValueError(f"{what} has no forward-mode derivative: detach its inputs")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no autograd of its own: call it under torch.no_grad(), or detach its inputs")


def _rows(t: Tensor) -> tuple[Tensor, int]:
    """``t``'s rows in memory, with unit column stride, and their pitch.

    Rows at any pitch are read where they are (as ``[rows, columns]``; a
    contiguous tensor keeps its shape); other orders are copied."""

    columns = t.shape[-1]
    if t.is_contiguous():
        return t, columns
    if t.ndim != 2:
        t = t.reshape(-1, columns)
        if t.is_contiguous():
            return t, columns
    rows = t.shape[0]
    if columns > 1 and t.stride(1) != 1:
        t = t.contiguous()
    pitch = t.stride(0) if rows > 1 else columns
    if pitch < columns:   # expanded rows
        t = t.contiguous()
        pitch = columns
    return t, pitch


def _new_values(lead: tuple[int, ...], columns: int, device: torch.device) -> tuple[Tensor, int]:
    pitch = (columns + 15) & ~15
    store = torch.empty(*lead, pitch, dtype=torch.int8, device=device)
    return (store if pitch == columns else store[..., :columns]), pitch


def _values_rows(t: Tensor) -> tuple[Tensor, int]:
    """8-bit rows as the kernels read them: 16-byte aligned at a pitch of a
    multiple of 16, with the last row's last 16 bytes inside the storage."""

    columns = t.shape[-1]
    if not (columns | t.data_ptr()) & 15 and t.is_contiguous():
        return t, columns
    rows = t.numel() // columns
    t, pitch = _rows(t)
    if rows == 1:
        pitch = (columns + 15) // 16 * 16
    fits = pitch % 16 == 0 and t.data_ptr() % 16 == 0
    if fits and columns % 16 and rows:
        last = t.storage_offset() + (rows - 1) * pitch + (columns + 15) // 16 * 16
        fits = last <= t.untyped_storage().nbytes()
    if not fits:
        padded, pitch = _new_values((rows,), columns, t.device)
        padded.copy_(t.reshape(rows, columns))
        t = padded
    return t, pitch


def _check_quantized(what: str, rows: QuantizedRows, device: torch.device | None = None) -> None:
    values, scales, group = rows
    if values.dtype is not _INT8 or scales.dtype is not _FLOAT32:
        raise ValueError(f"{what}: quantized rows are int8 values with fp32 scales")
    if group is not None and group != INT8_GROUP:
        raise NotImplementedError(f"{what}: a scale for each row (group None) or each {INT8_GROUP} columns")
    shape = values.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: expected rows of at least one column, got shape {tuple(shape)}")
    *lead, columns = shape
    if scales.shape != (*lead, 1 if group is None else -(-columns // group)):
        raise ValueError(f"{what}: scales of shape {tuple(scales.shape)} do not fit values of shape {tuple(shape)}")
    if not values.is_cuda:
        raise ValueError(f"{what}: HIP kernels require tensors on a ROCm device")
    index = values.get_device() if device is None else device.index
    if scales.get_device() != index or values.get_device() != index:
        raise ValueError(f"{what}: all tensors must be on one device")


def quantize_int8_hip(x: Tensor, group: int | None = None) -> QuantizedRows:
    """``x``'s rows (the last dimension; fp32, fp16 or bf16) in 8 bits.

    ``scale = max(amax, 127 * 2^-126) / 127`` over each row (``group`` None, up
    to 65536 columns: tokens and output channels of ``linear_int8_hip``) or
    each 128 columns of it (``INT8_GROUP``: saved activations), values
    ``round(x / scale)`` with fp32's division (the scale is amax times the fp32
    number nearest to 1 / 127).  A row (group) with an infinity or a NaN stands
    for NaN throughout.
    """

    what = "quantize_int8_hip"
    _no_grad(what, x)
    code = _check_input(what, x, _CODES)
    if group is not None and group != INT8_GROUP:
        raise NotImplementedError(f"{what}: a scale for each row (group None) or each {INT8_GROUP} columns")
    device = x.device
    *lead, columns = x.shape
    rows, pitch = _rows(x)
    values, ldv = _new_values(lead, columns, device)
    groups = 1 if group is None else -(-columns // INT8_GROUP)
    scales = torch.empty(*lead, groups, dtype=_FLOAT32, device=device)
    _launch(what, device, _lib.get().da_quantize_int8, rows.data_ptr(), x.numel() // columns, columns, pitch, code, group or 0,
            values.data_ptr(), ldv, scales.data_ptr())
    return QuantizedRows(values, scales, group)


def dequantize_int8_hip(rows: QuantizedRows, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """What the 8-bit rows stand for: ``values * scale``, rounded once to ``dtype``."""

    what = "dequantize_int8_hip"
    _no_grad(what, rows[1])
    _check_quantized(what, rows)
    values, scales, group = rows
    code = dtype_code(dtype)
    device = values.device
    out = torch.empty(*values.shape, dtype=dtype, device=device)
    values, pitch = _values_rows(values)
    scales = scales.contiguous()
    columns = values.shape[-1]
    _launch(what, device, _lib.get().da_dequantize_int8, values.data_ptr(), values.numel() // columns, columns, pitch,
            scales.data_ptr(), group or 0, out.data_ptr(), columns, code)
    return out


def linear_int8_hip(
    x: Tensor | QuantizedRows,
    weight: QuantizedRows,
    bias: Tensor | None = None,
    *,
    activation: str | None = None,
    residual: Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> Tensor:
    """``act(x @ weight.T (+ bias)) (+ residual)`` on 8-bit integers.

    ``weight``: ``quantize_int8_hip`` of the ``[out_features, in_features]``
    matrix (a scale for each output channel), made once.  ``x``: 8-bit rows
    with a scale for each token (``add_rms_norm_int8_hip``), or a 16-bit
    tensor, which is quantized so here.  The products and sums are exact
    integers; scales, bias and ``activation`` (None or ``"gelu"``) are fp32,
    the result is rounded to ``dtype`` (default: the 16-bit input's or
    residual's type, else bf16), then the residual is added and rounded, as by
    ``linear_hip``.  For inference: no backward.
    """

    what = "linear_int8_hip"
    if activation is not None and activation != "gelu":
        raise ValueError(f"unsupported activation {activation!r}")
    if isinstance(x, QuantizedRows):
        _check_quantized(what, x)
        x, x_scales, group = x
        if group is not None:
            raise ValueError(f"{what}: x needs one scale for each token")
        x_code = _lib.DA_I8
        if dtype is None:
            dtype = torch.bfloat16 if residual is None else residual.dtype
    else:
        x_scales = None
        x_code = _check_input(what, x)
        if dtype is None:
            dtype = x.dtype
    shape, device = x.shape, x.device
    _check_quantized(what, weight, device)
    w, w_scales, group = weight
    if group is not None or w.ndim != 2:
        raise ValueError(f"{what}: the weight is [out_features, in_features] with one scale for each output channel")
    code = _HALF_CODES.get(dtype)
    if code is None:
        raise ValueError(f"{what}: the output must be fp16 or bf16, not {dtype}")
    out_features, in_features = w.shape
    if shape[-1] != in_features:
        raise ValueError(f"{what}: rows of {shape[-1]} columns against a weight of {in_features}")
    *lead, _ = shape
    out_shape = (*lead, out_features)
    _no_grad(what, x, x_scales, w_scales, bias, residual)
    bias_ptr, bias_code = None, _lib.DA_F32
    if bias is not None:
        bias_code = _check_param(what, device, bias, out_features)
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    res_ptr, ldr = None, 0
    if residual is not None:
        if residual.shape != out_shape or residual.dtype is not dtype:
            raise ValueError(f"{what}: the residual must match the output's shape and dtype")
        _check_on(what, device, residual)
        residual, ldr = _rows(residual)
        res_ptr = residual.data_ptr()
    lib = _lib.get()
    w, ldw = _values_rows(w)
    w_scales = w_scales.contiguous()
    scales_ptr, workspace_ptr, nbytes = None, None, 0
    tokens = x.numel() // in_features
    if x_scales is None:
        rows, ldx = _rows(x)
        nbytes = lib.da_linear_int8_workspace_bytes(tokens, in_features, out_features, x_code, code)
        if nbytes:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
            workspace_ptr = workspace.data_ptr()
    else:
        rows, ldx = _values_rows(x)
        x_scales = x_scales.contiguous()
        scales_ptr = x_scales.data_ptr()
    out = torch.empty(*out_shape, dtype=dtype, device=device)
    _launch(what, device, lib.da_linear_int8, rows.data_ptr(), x_code, ldx, scales_ptr, tokens, in_features,
            w.data_ptr(), ldw, w_scales.data_ptr(), out_features, bias_ptr, bias_code,
            _lib.DA_ACT_GELU if activation else _lib.DA_ACT_NONE, res_ptr, ldr, out.data_ptr(), code, workspace_ptr, nbytes)
    return out


def _add_rms_norm(what, x, residual, weight, eps, want_out, want_int8):
    code = _check_input(what, x)
    shape, device, dtype = x.shape, x.device, x.dtype
    *lead, width = shape
    rows, ldx = _rows(x)
    total, res_ptr, ldr, total_ptr = x, None, 0, None
    if residual is not None:
        _check_like(what, x, residual)
        residual, ldr = _rows(residual)
        res_ptr = residual.data_ptr()
        total = torch.empty(*shape, dtype=dtype, device=device)
        total_ptr = total.data_ptr()
    weight_ptr, weight_code = None, _lib.DA_F32
    if weight is not None:
        weight_code = _check_param(what, device, weight, width)
        weight = weight.contiguous()
        weight_ptr = weight.data_ptr()
    out = values = scales = out_ptr = values_ptr = scales_ptr = None
    ldv = 0
    if want_out:
        out = torch.empty(*shape, dtype=dtype, device=device)
        out_ptr = out.data_ptr()
    if want_int8:
        values, ldv = _new_values(lead, width, device)
        scales = torch.empty(*lead, 1, dtype=_FLOAT32, device=device)
        values_ptr, scales_ptr = values.data_ptr(), scales.data_ptr()
    _launch(what, device, _lib.get().da_add_rms_norm, rows.data_ptr(), ldx, res_ptr, ldr, x.numel() // width, width, weight_ptr,
            weight_code, float(eps), code, total_ptr, out_ptr, values_ptr, ldv, scales_ptr)
    return out, values, scales, total


class _AddRmsNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):  # type: ignore[override]
        out, _, _, total = _add_rms_norm("add_rms_norm_hip", x, residual, weight, eps, True, False)
        ctx.save_for_backward(total, weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return out if residual is None else (out, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, grad_sum=None):  # type: ignore[override]
        total, weight = ctx.saved_tensors
        wants_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        wants_weight = ctx.needs_input_grad[2]
        if grad is None:
            d_x, d_weight = grad_sum, None
        else:
            d_x, d_weight = add_rms_norm_backward_hip(total, grad, grad_sum, weight, ctx.eps, want_weight=wants_weight)
        d_x = d_x if wants_x else None
        return (d_x if ctx.needs_input_grad[0] else None, d_x if ctx.needs_input_grad[1] else None,
                d_weight if wants_weight else None, None)


def add_rms_norm_hip(
    x: Tensor, residual: Tensor | None = None, weight: Tensor | None = None, eps: float = 1e-6
) -> tuple[Tensor, Tensor]:
    """``(n, s)``: the sum ``s = x + residual`` (rounded to x's 16-bit type; x
    itself without a residual) and its root-mean-square norm
    ``n = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension (at most
    16384 wide), statistics in fp32 and one rounding; one launch.
    Differentiable in x, the residual and the weight, through both outputs (in
    reverse mode; tensors with forward-mode tangents are refused).
    """

    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)) or (
        forward_ad._current_level >= 0 and _has_tangent(x, residual, weight)
    ):   # which has no forward-mode derivative, and says so
        got = _AddRmsNormFunction.apply(x, residual, weight, eps)
        return (got, x) if residual is None else got
    out, _, _, total = _add_rms_norm("add_rms_norm_hip", x, residual, weight, eps, True, False)
    return out, total


def add_rms_norm_int8_hip(
    x: Tensor, residual: Tensor | None = None, weight: Tensor | None = None, eps: float = 1e-6
) -> tuple[QuantizedRows, Tensor]:
    """``add_rms_norm_hip`` with its norm in 8 bits, a scale for each row: the
    fp32 norm is quantized without a rounding to 16 bits in between, by one
    multiplication (a value within fp32's roundings of a half of a step may
    become either neighbour).  The sum stays 16-bit.  For inference: no backward."""

    what = "add_rms_norm_int8_hip"
    _no_grad(what, x, residual, weight)
    _, values, scales, total = _add_rms_norm(what, x, residual, weight, eps, False, True)
    return QuantizedRows(values, scales), total


def add_rms_norm_backward_hip(
    total: Tensor,
    grad: Tensor,
    grad_sum: Tensor | None,
    weight: Tensor | None,
    eps: float = 1e-6,
    *,
    want_weight: bool = True,
) -> tuple[Tensor, Tensor | None]:
    """The backward of ``add_rms_norm_hip``: ``(grad_x, grad_weight)`` from its
    sum, the gradient at its norm and the one at its sum (None: zero).  grad_x
    is the gradient at x and at the residual; grad_weight (None without a
    weight, or unless wanted) is summed in fp32 in an order that the sizes
    fix, and rounded once to the weight's type.
    """

    what = "add_rms_norm_backward_hip"
    _no_grad(what, total, grad, grad_sum, weight)
    code = _check_input(what, total)
    _check_like(what, total, grad)
    shape, device = total.shape, total.device
    width = shape[-1]
    count = total.numel() // width
    lib = _lib.get()
    s, lds = _rows(total)
    g, ldg = _rows(grad)
    gs_ptr, ldgs = None, 0
    if grad_sum is not None:
        _check_like(what, total, grad_sum)
        grad_sum, ldgs = _rows(grad_sum)
        gs_ptr = grad_sum.data_ptr()
    grad_x = torch.empty(*shape, dtype=total.dtype, device=device)
    weight_ptr, weight_code = None, _lib.DA_F32
    grad_weight = grad_weight_ptr = workspace_ptr = None
    nbytes = 0
    if weight is not None:
        weight_code = _check_param(what, device, weight, width)
        weight = weight.contiguous()
        weight_ptr = weight.data_ptr()
        if want_weight:
            grad_weight = torch.empty(width, dtype=weight.dtype, device=device)
            grad_weight_ptr = grad_weight.data_ptr()
            nbytes = lib.da_add_rms_norm_backward_workspace_bytes(count, width)
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
            workspace_ptr = workspace.data_ptr()
    _launch(what, device, lib.da_add_rms_norm_backward, s.data_ptr(), lds, g.data_ptr(), ldg, gs_ptr, ldgs, count,
            width, weight_ptr, weight_code, float(eps), code, grad_x.data_ptr(), grad_weight_ptr, workspace_ptr, nbytes)
    return grad_x, grad_weight


def gelu_int8_hip(z: Tensor) -> tuple[Tensor, QuantizedRows]:
    """``(gelu(z), kept)``: the exact GELU of a 16-bit tensor, and z in 8 bits
    in groups of 128 for ``gelu_int8_backward_hip``, in one pass.  The output
    is of z itself; only the backward sees the kept rows."""

    what = "gelu_int8_hip"
    code = _check_input(what, z)
    _no_grad(what, z)
    shape, device = z.shape, z.device
    *lead, columns = shape
    rows, pitch = _rows(z)
    out = torch.empty(*shape, dtype=z.dtype, device=device)
    values, ldv = _new_values(lead, columns, device)
    scales = torch.empty(*lead, -(-columns // INT8_GROUP), dtype=_FLOAT32, device=device)
    _launch(what, device, _lib.get().da_gelu_int8, rows.data_ptr(), z.numel() // columns, columns, pitch, code, out.data_ptr(),
            values.data_ptr(), ldv, scales.data_ptr())
    return out, QuantizedRows(values, scales, INT8_GROUP)


def gelu_int8_backward_hip(kept: QuantizedRows, grad: Tensor, *, want_output: bool = True) -> tuple[Tensor, Tensor | None]:
    """``(grad_z, gelu)`` from the rows that ``gelu_int8_hip`` kept:
    ``grad * gelu'(zt)`` and, unless not wanted, ``gelu(zt)`` again (the
    operand of the next layer's weight gradient), with ``zt`` what the kept
    rows stand for; fp32, one rounding to grad's 16-bit type."""

    what = "gelu_int8_backward_hip"
    _no_grad(what, grad, kept[1])
    code = _check_input(what, grad)
    shape, device = grad.shape, grad.device
    _check_quantized(what, kept, device)
    values, scales, group = kept
    if group is None:
        raise ValueError(f"{what}: rows kept in groups of {INT8_GROUP} columns")
    if values.shape != shape:
        raise ValueError(f"{what}: gradients of shape {tuple(shape)} at kept rows of shape {tuple(values.shape)}")
    values, ldv = _values_rows(values)
    scales = scales.contiguous()
    g, ldg = _rows(grad)
    grad_z = torch.empty(*shape, dtype=grad.dtype, device=device)
    out = torch.empty(*shape, dtype=grad.dtype, device=device) if want_output else None
    columns = shape[-1]
    _launch(what, device, _lib.get().da_gelu_int8_backward, values.data_ptr(), values.numel() // columns, columns, ldv,
            scales.data_ptr(), g.data_ptr(), ldg, code, grad_z.data_ptr(), None if out is None else out.data_ptr())
    return grad_z, out
