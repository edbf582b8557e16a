"""The 8-bit operators against plain 64-bit forms.

Tolerances count roundings: half a step of the 16-bit output
(``torch.finfo(t).eps / 2`` of the value, and half the least subnormal), plus
the fp32 arithmetic's, bounded term by term beside each test.  The GELU's erf
is Abramowitz & Stegun 7.1.26, at most 1.5e-7 off, evaluated in fp32: 1e-6 in
all.
"""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

import double_attention as da
from double_attention import _lib, int8_ops

HALF = [torch.bfloat16, torch.float16]
F32 = 2.0 ** -24   # half a step of fp32
WIDTHS = [1, 7, 8, 9, 127, 128, 129, 135, 505, 512, 1001, 1536, 2049]


def _device() -> torch.device:
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    if not da.HIP_AVAILABLE:
        raise RuntimeError("HIP library not built; run python double-attention_amd/build.py")
    return torch.device("cuda")


def _randn(*shape, seed=0, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * spread
    x[..., :: 17] *= 6.0   # a few large channels
    return x.to(dtype).to(_device())


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the least subnormal: the rounding of values below the normal range."""

    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, expected, tolerance):
    off = (got.double() - expected).abs()
    worst = (off - tolerance).max().item() if off.numel() else 0.0
    assert not math.isnan(worst) and worst <= 0, f"off by {off.max().item():.3e}, {worst:.3e} more than allowed"


def groups_of(x, group):
    """``[..., groups, columns]`` of rows, zeros behind the last column."""

    if group is None:
        return x.unsqueeze(-2)
    n = -(-x.shape[-1] // group)
    padded = x.new_zeros(*x.shape[:-1], n * group)
    padded[..., : x.shape[-1]] = x
    return padded.view(*x.shape[:-1], n, group)


def check_kept(kept, x64, group, extra=0.0):
    """Scales and values of rows of 64-bit numbers, which the kernel may have
    had with a relative error of ``extra``."""

    parts = groups_of(x64, group)
    amax = parts.abs().amax(-1)
    expected = torch.clamp(amax, min=127 * 2.0 ** -126) / 127
    # amax itself is exact; one product with the rounded 1/127.
    close(kept.scales, expected, expected * (3 * F32 + extra))
    stands = groups_of(kept.values.double(), group) * kept.scales.double().unsqueeze(-1)
    # Half a step, and the fp32 product's error of at most 127 steps * 4 F32.
    close(stands, parts, kept.scales.double().unsqueeze(-1) * (0.5 + 127 * (4 * F32 + extra)) + extra * parts.abs())
    assert kept.values.abs().max().item() <= 127 if kept.values.numel() else True


@pytest.mark.gpu
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("dtype", [*HALF, torch.float32])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize(width, dtype, group) -> None:
    for rows in (1, 5, 67):
        x = _randn(rows, width, seed=width, dtype=dtype)
        kept = da.quantize_int8_hip(x, group)
        assert kept.values.shape == x.shape and kept.values.dtype == torch.int8
        check_kept(kept, x.double(), group)
        for out_type in (*HALF, torch.float32):
            back = da.dequantize_int8_hip(kept, out_type)
            exact = groups_of(kept.values.double(), group) * kept.scales.double().unsqueeze(-1)
            exact = exact.flatten(-2)[..., :width]
            close(back, exact, exact.abs() * (half_step(out_type) + F32) + least(out_type))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [4096, 4097, 8192, 16384, 16391, 32768, 65535, 65536])
def test_quantize_wide_rows(width, dtype) -> None:
    x = _randn(3, width, seed=1, dtype=dtype)
    check_kept(da.quantize_int8_hip(x), x.double(), None)
    check_kept(da.quantize_int8_hip(x, 128), x.double(), 128)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [None, 128])
def test_quantize_layouts(group) -> None:
    """Rows at other pitches, offsets and orders, and leading dimensions."""

    base = _randn(40, 700, seed=2, dtype=torch.bfloat16)
    views = [base[:, 3:303], base[::2, 5:261], base.t()[:, :33], base[3, :300], base.view(4, 10, 700)[:, ::3, 1:258],
             base[:1].expand(6, 700), base[:0], base.view(4, 10, 700)]
    for x in views:
        kept = da.quantize_int8_hip(x, group)
        same = da.quantize_int8_hip(x.contiguous(), group)
        assert kept.values.shape == x.shape and torch.equal(kept.values, same.values)
        assert torch.equal(kept.scales, same.scales)
        assert torch.equal(da.dequantize_int8_hip(kept), da.dequantize_int8_hip(same))
    # Kept rows that are not at the kernels' pitch.
    kept = da.quantize_int8_hip(base, group)
    loose = da.QuantizedRows(kept.values.contiguous()[:, :], kept.scales, group)
    assert torch.equal(da.dequantize_int8_hip(loose), da.dequantize_int8_hip(kept))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [None, 128])
@pytest.mark.parametrize("dtype", [*HALF, torch.float32])
def test_quantize_values_out_of_the_ordinary(dtype, group) -> None:
    x = _randn(8, 300, seed=3, dtype=dtype)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 130] = float("nan")
    x[3, 299] = -float("inf")
    x[4] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps   # the least subnormal
    x[5] = torch.finfo(dtype).max
    x[6] = -0.0
    x[7, :] = 0
    x[7, 150] = -3.0
    kept = da.quantize_int8_hip(x, group)
    bad = ~torch.isfinite(groups_of(x, group)).all(-1)
    assert torch.equal(torch.isnan(kept.scales), bad)
    assert (groups_of(kept.values, group)[bad] == 0).all()
    good = ~bad
    parts = groups_of(x.double(), group)[good]
    scales = kept.scales[good].double()
    assert (scales >= 2.0 ** -126).all()
    stands = groups_of(kept.values.double(), group)[good] * scales.unsqueeze(-1)
    close(stands, parts, scales.unsqueeze(-1) * (0.5 + 127 * 4 * F32))
    back = da.dequantize_int8_hip(kept, torch.float32)
    assert torch.equal(torch.isnan(groups_of(back, group)).any(-1), bad)
    assert (back[0] == 0).all() and (back[6] == 0).all()


def halves(rows, width, dtype):
    """Rows with both halves of their largest magnitude, 63.5 steps but for the scale's rounding."""

    x = _randn(rows, width, seed=5, dtype=dtype)
    x[:, ::16] = x[:, 1::16] = 0
    amax = x.abs().amax(-1, keepdim=True)
    x[:, :1], x[:, 16::16], x[:, 1::16] = amax, amax / 2, -amax / 2
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [*HALF, torch.float32])
def test_quantize_rounds_the_quotient(dtype) -> None:
    """The integers are those of fp32's division, ties to even, whatever forms them."""

    x = halves(300, 320, dtype)
    x[200:] *= 2.0 ** -8
    # Scales without a rounding: every odd multiple of amax / 254 is half a step.
    exact = torch.arange(-127, 128, dtype=torch.float64) / 127
    for row, j in enumerate([1, 2, 3, 5, 7, 8, 9, 11, 13, 15] if dtype == torch.float16 else [1, 2]):
        x[row] = 0
        x[row, :255] = (127 * j * exact).to(dtype)
        x[row, 256:290] = torch.arange(34, dtype=dtype) * (j / 2)
        x[row, 290] = -127 * j
    kinds = [da.quantize_int8_hip(x), da.quantize_int8_hip(x, 128)]
    if dtype != torch.float32:
        kinds.append(da.gelu_int8_hip(x)[1])
    for kept in kinds:
        scales = kept.scales.cpu().repeat_interleave(128 if kept.group else 320, 1)[:, :320]
        assert torch.equal(kept.values.cpu().float(), torch.round(x.cpu().float() / scales))
    if dtype != torch.float32:
        # Tokens that are quantized where they are multiplied: few, and in tiles.
        w = da.quantize_int8_hip(_randn(300, 320, seed=6))
        for rows in (1, 16, 300):
            kept = da.quantize_int8_hip(x[:rows])
            assert torch.equal(da.linear_int8_hip(x[:rows], w), da.linear_int8_hip(kept, w, dtype=dtype))


def linear64(kept_x, kept_w, bias, gelu):
    """The layer's result before its rounding, and the fp32 error bound."""

    product = kept_x.values.double().flatten(0, -2) @ kept_w.values.double().t()
    product *= kept_x.scales.double().reshape(-1, 1) * kept_w.scales.double().reshape(1, -1)
    b = torch.zeros_like(product[0]) if bias is None else bias.double()
    y = product + b
    # Integer to fp32, two scales, one addition.
    error = 4 * F32 * (product.abs() + b.abs())
    if gelu:
        # |gelu'| <= 1.13; erf 1e-6 off; the product's roundings.
        error = 1.13 * error + 0.5e-6 * y.abs() + 4 * F32 * y.abs()
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    return y, error


def check_linear(got, kept_x, kept_w, bias, gelu, residual, dtype):
    y, error = linear64(kept_x, kept_w, bias, gelu)
    error = error + y.abs() * half_step(dtype) + least(dtype)
    if residual is not None:
        y = y + residual.double().reshape(y.shape)
        error = error + (y.abs() + error) * half_step(dtype) + least(dtype)
    close(got.reshape(y.shape), y, error)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(("rows", "inner", "outer"), [
    (1, 512, 1536), (1, 1, 1), (2, 16, 4), (3, 17, 9), (5, 127, 33), (16, 128, 130), (17, 129, 128), (31, 1000, 65),
    (33, 64, 257), (64, 1536, 512), (65, 100, 64), (127, 255, 127), (128, 256, 128), (129, 384, 129),
    (300, 1000, 1111), (513, 512, 1536), (1, 4096, 4096), (16, 4096, 1000), (48, 2048, 640), (4, 65536, 24),
    (700, 700, 3), (2000, 15, 300), (2100, 200, 1500), (1500, 130, 1900), (3000, 64, 2000), (4100, 333, 2500), (5000, 700, 4500),
    (200, 512, 200), (130, 513, 70), (66, 1024, 65), (700, 900, 1500), (4000, 100, 4000), (4000, 200, 4000), (4000, 300, 4000), (3300, 50, 2100), (2000, 100, 1300), (2000, 200, 1300),
    (90, 1025, 64), (40, 1537, 40), (1100, 500, 1500), (4000, 33, 500),
])
def test_linear(rows, inner, outer, dtype) -> None:
    x = _randn(rows, inner, seed=rows, dtype=dtype)
    weight = _randn(outer, inner, seed=outer, spread=inner ** -0.5)
    w = da.quantize_int8_hip(weight)
    kept = da.quantize_int8_hip(x)
    bias = _randn(outer, seed=5, dtype=torch.float32)
    residual = _randn(rows, outer, seed=6, dtype=dtype)
    for b, gelu, res in ((None, False, None), (bias, True, None), (bias.to(dtype), False, residual), (None, True, residual)):
        options = {"activation": "gelu" if gelu else None, "residual": res}
        got = da.linear_int8_hip(x, w, b, **options)
        assert got.dtype == dtype and got.shape == (rows, outer)
        check_linear(got, kept, w, b, gelu, res, dtype)
        again = da.linear_int8_hip(kept, w, b, dtype=dtype, **options)
        assert torch.equal(got, again), "16-bit rows and the same rows quantized before"
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    check_linear(da.linear_int8_hip(x, w, dtype=other), kept, w, None, False, None, other)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("inner", [8, 511, 513, 1024, 2047, 2049, 3583, 4095])
@pytest.mark.parametrize("rows", [1, 7, 8, 9, 15, 16])
def test_linear_few_tokens_of_any_width(rows, inner, dtype) -> None:
    """One or two tokens a wave, whole and partial passes over them."""

    x = _randn(rows + 3, inner + 5, seed=inner + rows, dtype=dtype)[2:-1, 3:-2]
    w = da.quantize_int8_hip(_randn(37, inner, seed=1, spread=inner ** -0.5))
    kept = da.quantize_int8_hip(x)
    got = da.linear_int8_hip(x, w)
    check_linear(got, kept, w, None, False, None, dtype)
    assert torch.equal(got, da.linear_int8_hip(kept, w, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("inner", [1, 3, 5, 7, 9, 1023])
@pytest.mark.parametrize(("rows", "outer"), [(13, 7), (100, 64), (3900, 500), (5000, 2100)])
def test_linear_narrow_and_odd_tokens(rows, outer, inner, dtype) -> None:
    """Tokens of less than a chunk, and of one that ends inside a chunk."""

    x = _randn(rows + 1, inner + 3, seed=inner, dtype=dtype)[:-1, 1:-2]
    w = da.quantize_int8_hip(_randn(outer, inner, seed=1, spread=inner ** -0.5))
    kept = da.quantize_int8_hip(x)
    got = da.linear_int8_hip(x, w)
    check_linear(got, kept, w, None, False, None, dtype)
    assert torch.equal(got, da.linear_int8_hip(kept, w, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [70, 96, 200])
def test_rows_of_three_dimensions(width) -> None:
    """The rows of [a, b, width] tensors are those of [a b, width] ones."""

    x = _randn(3, 5, width, seed=1, dtype=torch.bfloat16)
    flat = x.view(15, width)
    weight = _randn(width, seed=2, dtype=torch.bfloat16)
    w = da.quantize_int8_hip(_randn(24, width, seed=3))
    for group in (None, 128):
        kept, same = da.quantize_int8_hip(x, group), da.quantize_int8_hip(flat, group)
        assert torch.equal(kept.values.flatten(0, 1), same.values) and torch.equal(kept.scales.flatten(0, 1), same.scales)
        assert torch.equal(da.dequantize_int8_hip(kept).flatten(0, 1), da.dequantize_int8_hip(same))
        turned = da.QuantizedRows(kept.values.transpose(0, 1), kept.scales.transpose(0, 1), group)
        assert torch.equal(da.dequantize_int8_hip(turned), da.dequantize_int8_hip(kept).transpose(0, 1))
        if group is None:
            assert torch.equal(da.linear_int8_hip(kept, w).flatten(0, 1), da.linear_int8_hip(same, w))
            assert torch.equal(da.linear_int8_hip(turned, w), da.linear_int8_hip(kept, w).transpose(0, 1))
        else:
            for a, b in zip(da.gelu_int8_backward_hip(kept, x), da.gelu_int8_backward_hip(same, flat)):
                assert torch.equal(a.flatten(0, 1), b)
    for a, b in zip(da.add_rms_norm_hip(x, x, weight), da.add_rms_norm_hip(flat, flat, weight)):
        assert torch.equal(a.flatten(0, 1), b)
    a, b = (da.add_rms_norm_backward_hip(t, t, t, weight) for t in (x, flat))
    assert torch.equal(a[0].flatten(0, 1), b[0]) and torch.equal(a[1], b[1])
    a, b = da.add_rms_norm_backward_hip(x.transpose(0, 1), x.transpose(0, 1), None, weight), da.add_rms_norm_backward_hip(
        x.transpose(0, 1).contiguous(), x.transpose(0, 1).contiguous(), None, weight)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize(("rows", "inner", "outer"), [(1, 70, 90), (40, 70, 90), (200, 200, 300), (2100, 1100, 1300)])
def test_linear_any_bytes(rows, inner, outer) -> None:
    """Integers of the whole range, -128 too, and anything behind the rows' columns."""

    device = _device()
    g = torch.Generator().manual_seed(rows)

    def rows_of(n):
        store = torch.randint(-128, 128, (n, (inner + 15) // 16 * 16 + 16), generator=g, dtype=torch.int8).to(device)
        scales = (0.5 + torch.rand(n, 1, generator=g)).to(device) * 1e-3
        return da.QuantizedRows(store[:, :inner], scales)

    x, w = rows_of(rows), rows_of(outer)
    x.values[0], w.values[0] = -128, -128
    got = da.linear_int8_hip(x, w, dtype=torch.float16)
    check_linear(got, x, w, None, False, None, torch.float16)
    # Rows at no such pitch, a transposed weight, tokens in reverse order.
    loose = da.QuantizedRows(x.values.contiguous(), x.scales)
    turned = da.QuantizedRows(w.values.t().contiguous().t(), w.scales)
    assert torch.equal(da.linear_int8_hip(loose, turned, dtype=torch.float16), got)
    back = da.QuantizedRows(x.values.flip(0)[:, :inner], x.scales.flip(0))
    assert torch.equal(da.linear_int8_hip(back, w, dtype=torch.float16), got.flip(0))


@pytest.mark.gpu
def test_linear_leading_dimensions_and_strided_operands() -> None:
    x = _randn(3, 5, 96, seed=1, dtype=torch.bfloat16)
    w = da.quantize_int8_hip(_randn(40, 96, seed=2))
    residual = _randn(3, 5, 47, seed=3, dtype=torch.bfloat16)[..., 7:]
    got = da.linear_int8_hip(x, w, residual=residual)
    flat = da.linear_int8_hip(x.view(15, 96), w, residual=residual.reshape(15, 40))
    assert got.shape == (3, 5, 40) and torch.equal(got.view(15, 40), flat)
    assert torch.equal(da.linear_int8_hip(x.transpose(0, 1), w), da.linear_int8_hip(x, w).transpose(0, 1))
    assert torch.equal(da.linear_int8_hip(x[1, 2], w), da.linear_int8_hip(x, w)[1, 2])
    assert da.linear_int8_hip(x[:0], w).shape == (0, 5, 40)
    wide = _randn(64, 96 * 3 + 5, seed=4, dtype=torch.bfloat16)
    assert torch.equal(da.linear_int8_hip(wide[:, 96:192], w), da.linear_int8_hip(wide[:, 96:192].contiguous(), w))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_linear_tokens_without_integers(rows) -> None:
    """A token that holds an infinity or a NaN is NaN in every feature, and no
    other token is touched."""

    x = _randn(rows, 200, seed=7, dtype=torch.bfloat16)
    w = da.quantize_int8_hip(_randn(130, 200, seed=8))
    clean = da.linear_int8_hip(x, w)
    x[0, 3], x[rows - 1, 199] = float("nan"), float("inf")
    got = da.linear_int8_hip(x, w)
    assert torch.isnan(got[0]).all() and torch.isnan(got[rows - 1]).all()
    assert torch.equal(got[1 : rows - 1], clean[1 : rows - 1])


NORM_F32 = 48 * F32   # the sum of squares: at most 64 additions a thread, then a tree; halved by the root


def norm64(s, w, eps):
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    return s * rstd * (1.0 if w is None else w), rstd


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("width", [*WIDTHS, 1018, 1024, 4096, 8191, 16377, 16383, 16384])
def test_add_rms_norm(width, dtype) -> None:
    for rows in (1, 6, 131):
        x = _randn(rows, width, seed=width, dtype=dtype)
        residual = _randn(rows, width, seed=rows, dtype=dtype, spread=3.0)
        weight = 1 + 0.3 * _randn(width, seed=9)
        for r, w in ((residual, weight.to(dtype)), (None, weight), (residual, None)):
            total = x if r is None else (x.float() + r.float()).to(dtype)
            n, _ = norm64(total.double(), None if w is None else w.double(), 1e-5)
            out, s = da.add_rms_norm_hip(x, r, w, 1e-5)
            assert torch.equal(s, total)
            close(out, n, n.abs() * (half_step(dtype) + NORM_F32) + least(dtype))
            kept, s = da.add_rms_norm_int8_hip(x, r, w, 1e-5)
            assert torch.equal(s, total)
            check_kept(kept, n, None, NORM_F32)


@pytest.mark.gpu
def test_add_rms_norm_layouts_and_rows_out_of_the_ordinary() -> None:
    base = _randn(30, 600, seed=1, dtype=torch.bfloat16)
    weight = _randn(3 * 257, seed=2)[::3]
    for x, r in ((base[:, 1:258], base[:, 300:557]), (base[::3, :257], base[10:20, 9:266]),
                 (base.view(5, 6, 600)[:, :, :257], base.view(5, 6, 600)[..., 3:260]), (base[4, :257], base[5, :257]),
                 (base[:7, :257], base[:1, :257].expand(7, 257)), (base[:0, :257], base[:0, :257])):
        want, total = da.add_rms_norm_hip(x.contiguous(), r.contiguous(), weight.contiguous())
        got, s = da.add_rms_norm_hip(x, r, weight)
        assert torch.equal(got, want) and torch.equal(s, total) and got.shape == x.shape
        a, _ = da.add_rms_norm_int8_hip(x, r, weight)
        b, _ = da.add_rms_norm_int8_hip(x.contiguous(), r.contiguous(), weight.contiguous())
        assert torch.equal(a.values, b.values) and torch.equal(a.scales, b.scales)
    x = _randn(5, 300, seed=3, dtype=torch.bfloat16)
    clean = da.dequantize_int8_hip(da.add_rms_norm_int8_hip(x)[0])
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 299] = float("inf")
    got = da.dequantize_int8_hip(da.add_rms_norm_int8_hip(x)[0])
    assert (got[0] == 0).all() and torch.isnan(got[1]).all() and torch.isnan(got[2]).all()
    assert torch.equal(got[3:], clean[3:])
    # A tiny eps: the inverse scale of an all-zero row is beyond fp32.
    assert (da.add_rms_norm_int8_hip(x[:1], eps=1e-30)[0].values == 0).all()
    assert (da.add_rms_norm_hip(x[:1], eps=1e-30)[0] == 0).all()


def backward64(s, g, gs, w, eps):
    """Gradients of ``<n, g> + <s, gs>`` and the sums of their terms' magnitudes."""

    _, rstd = norm64(s, None, eps)
    xh = s * rstd
    gw = g if w is None else g * w
    d = rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True)) + (0.0 if gs is None else gs)
    size = rstd * (gw.abs() + xh.abs() * (gw * xh).abs().mean(-1, keepdim=True)) + (0.0 if gs is None else gs.abs())
    return d, size, (g * xh).sum(0), (g * xh).abs().sum(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("width", [*WIDTHS, 1018, 1024, 4096, 8191, 16377, 16383, 16384])
def test_add_rms_norm_backward(width, dtype) -> None:
    for rows in (1, 6, 700):
        s = _randn(rows, width, seed=width, dtype=dtype)
        g = _randn(rows, width, seed=rows, dtype=dtype)
        gs = _randn(rows, width, seed=rows + 1, dtype=dtype)
        weight = 1 + 0.3 * _randn(width, seed=9)
        for w, extra in ((weight.to(dtype), gs), (weight, None), (None, gs)):
            d, size, dw, dw_size = backward64(s.double(), g.double(), None if extra is None else extra.double(),
                                              None if w is None else w.double(), 1e-5)
            grad_x, grad_weight = da.add_rms_norm_backward_hip(s, g, extra, w, 1e-5)
            # 8 roundings a term besides the two sums'.
            close(grad_x, d, d.abs() * half_step(dtype) + size * (2 * NORM_F32 + 8 * F32) + least(dtype))
            if w is None:
                assert grad_weight is None
                continue
            assert grad_weight.dtype == w.dtype
            # A thread's rows, then the workgroups' sums: at most rows + 32 additions.
            bound = dw_size * ((rows + 32) * F32 + NORM_F32 + 2 * F32)
            close(grad_weight, dw, dw.abs() * half_step(w.dtype) + bound + least(w.dtype))
            again = da.add_rms_norm_backward_hip(s, g, extra, w, 1e-5)
            assert torch.equal(grad_x, again[0]) and torch.equal(grad_weight, again[1])


@pytest.mark.gpu
def test_add_rms_norm_backward_no_rows_and_no_weight_gradient() -> None:
    s = _randn(4, 40, seed=1, dtype=torch.bfloat16)
    weight = _randn(40, seed=2)
    grad_x, grad_weight = da.add_rms_norm_backward_hip(s[:0], s[:0], None, weight)
    assert grad_x.shape == (0, 40) and (grad_weight == 0).all()
    a, none = da.add_rms_norm_backward_hip(s, s, s, weight, want_weight=False)
    assert none is None and torch.equal(a, da.add_rms_norm_backward_hip(s, s, s, weight)[0])
    wide = _randn(4, 100, seed=3, dtype=torch.bfloat16)
    b, dw = da.add_rms_norm_backward_hip(wide[:, 1:41], wide[:, 50:90], wide[:, 7:47], weight)
    c, dw2 = da.add_rms_norm_backward_hip(wide[:, 1:41].contiguous(), wide[:, 50:90].contiguous(),
                                          wide[:, 7:47].contiguous(), weight)
    assert torch.equal(b, c) and torch.equal(dw, dw2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_add_rms_norm_autograd(dtype) -> None:
    """Through both outputs, one of them, shared inputs and no residual."""

    x0, r0 = _randn(2, 9, 130, seed=1, dtype=dtype), _randn(2, 9, 130, seed=2, dtype=dtype)
    w0 = 1 + 0.3 * _randn(130, seed=3)
    g, gs = _randn(2, 9, 130, seed=4, dtype=dtype), _randn(2, 9, 130, seed=5, dtype=dtype)

    def grads(use_n, use_s, residual, shared=False):
        x = x0.clone().requires_grad_()
        r = x if shared else r0.clone().requires_grad_() if residual else None
        w = w0.clone().requires_grad_()
        n, s = da.add_rms_norm_hip(x, r, w)
        loss = (n.float() * g.float()).sum() * use_n + (s.float() * gs.float()).sum() * use_s if use_n and use_s else \
            (n.float() * g.float()).sum() if use_n else (s.float() * gs.float()).sum()
        loss.backward()
        return s.detach(), x.grad, None if r is None or shared else r.grad, w.grad

    for use_n, use_s, residual in ((1, 1, True), (1, 0, True), (0, 1, True), (1, 1, False), (1, 0, False)):
        s, dx, dr, dw = grads(use_n, use_s, residual)
        if use_n:
            want, want_w = da.add_rms_norm_backward_hip(s, g, gs if use_s and residual else None, w0)
            if use_s and not residual:
                want = want + gs   # the sum is x itself: autograd adds
            assert torch.equal(dw, want_w)
        else:
            want = gs
            assert dw is None
        assert torch.equal(dx, want)
        assert dr is None or torch.equal(dr, want)
    s, dx, _, _ = grads(1, 1, True, shared=True)
    want, _ = da.add_rms_norm_backward_hip(s, g, gs, w0)
    assert torch.equal(dx, want + want)


def test_norm_gradient_formula_against_differences() -> None:
    g = torch.Generator().manual_seed(0)
    s, grad, gs = (torch.randn(3, 11, generator=g).double() for _ in range(3))
    w = torch.randn(11, generator=g).double()

    def loss(s, w):
        return (norm64(s, w, 1e-3)[0] * grad).sum() + (s * gs).sum()

    d, _, dw, _ = backward64(s, grad, gs, w, 1e-3)
    for where, got in ((s, d), (w, dw)):
        flat = where.view(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + 1e-5
            up = loss(s, w)
            flat[i] = keep - 1e-5
            down = loss(s, w)
            flat[i] = keep
            assert abs((up - down).item() / 2e-5 - got.reshape(-1)[i].item()) < 1e-7


def gelu64(z):
    below = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
    return z * below, below + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5


def test_gelu_slope_against_differences() -> None:
    z = torch.linspace(-8, 8, 4001, dtype=torch.float64)
    h = 1e-5
    assert ((gelu64(z + h)[0] - gelu64(z - h)[0]) / (2 * h) - gelu64(z)[1]).abs().max() < 1e-9


def check_gelu(z, grad, out, kept, grad_z, again):
    dtype = z.dtype
    u, _ = gelu64(z.double())
    close(out, u, u.abs() * half_step(dtype) + z.double().abs() * (0.5e-6 + 4 * F32) + least(dtype))
    check_kept(kept, z.double(), 128)
    zt = (groups_of(kept.values.double(), 128) * kept.scales.double().unsqueeze(-1)).flatten(-2)[..., : z.shape[-1]]
    u, slope = gelu64(zt)
    d = grad.double() * slope
    # q * scale is rounded once; erf, the density (its exponent rounded: at
    # most 0.4 * 3 F32) and the products' roundings.
    error = grad.double().abs() * (0.5e-6 + 8 * F32 * (1 + zt.abs()))
    close(grad_z, d, d.abs() * half_step(dtype) + error + least(dtype))
    close(again, u, u.abs() * half_step(dtype) + zt.abs() * (0.5e-6 + 6 * F32) + least(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("width", WIDTHS)
def test_gelu(width, dtype) -> None:
    for rows in (1, 5, 67):
        z = _randn(rows, width, seed=width, dtype=dtype, spread=1.5)
        grad = _randn(rows, width, seed=rows, dtype=dtype)
        out, kept = da.gelu_int8_hip(z)
        grad_z, again = da.gelu_int8_backward_hip(kept, grad)
        check_gelu(z, grad, out, kept, grad_z, again)
        only, none = da.gelu_int8_backward_hip(kept, grad, want_output=False)
        assert none is None and torch.equal(only, grad_z)


@pytest.mark.gpu
def test_gelu_layouts_and_rows_out_of_the_ordinary() -> None:
    base = _randn(24, 700, seed=1, dtype=torch.float16)
    grads = _randn(24, 700, seed=2, dtype=torch.float16)
    for z, g in ((base[:, 1:300], grads[:, 3:302]), (base[::2, :257], grads[12:, 5:262]),
                 (base.view(4, 6, 700)[..., :129], grads.view(4, 6, 700)[..., 9:138]), (base[2, :90], grads[1, :90]),
                 (base.t()[:, :13], grads.t()[:, 3:16]), (base[:3], grads[:1].expand(3, 700)), (base[:0], grads[:0])):
        out, kept = da.gelu_int8_hip(z)
        same, kept2 = da.gelu_int8_hip(z.contiguous())
        assert torch.equal(out, same) and torch.equal(kept.values, kept2.values) and torch.equal(kept.scales, kept2.scales)
        a, u = da.gelu_int8_backward_hip(kept, g)
        b, u2 = da.gelu_int8_backward_hip(kept2, g.contiguous())
        assert torch.equal(a, b) and torch.equal(u, u2) and a.shape == z.shape
    z = _randn(3, 300, seed=3, dtype=torch.bfloat16)
    z[0] = 0
    z[1, 200] = float("nan")
    z[2, 5] = 3e38
    out, kept = da.gelu_int8_hip(z)
    assert torch.isnan(out[1, 200]) and not torch.isnan(out[1, :200]).any() and out[2, 5] == z[2, 5]
    grad_z, again = da.gelu_int8_backward_hip(kept, torch.ones_like(z))
    assert (again[0] == 0).all() and (grad_z[0] == 0.5).all()
    assert torch.isnan(grad_z[1, 128:256]).all() and not torch.isnan(grad_z[1, :128]).any()
    assert grad_z[2, 5] == 1


@pytest.mark.gpu
def test_capture_other_streams_and_repeats() -> None:
    """The operators in a captured graph, replayed between eager work, and on
    another stream: the same bits every time."""

    x = _randn(70, 300, seed=1, dtype=torch.bfloat16)
    r = _randn(70, 300, seed=2, dtype=torch.bfloat16)
    weight = 1 + 0.1 * _randn(300, seed=3)
    w1 = da.quantize_int8_hip(_randn(500, 300, seed=4, spread=0.1))
    w2 = da.quantize_int8_hip(_randn(300, 500, seed=5, spread=0.1))
    grad = _randn(70, 500, seed=6, dtype=torch.bfloat16)

    def work():
        n, s = da.add_rms_norm_int8_hip(x, r, weight)
        z = da.linear_int8_hip(n, w1, dtype=torch.bfloat16)
        u, kept = da.gelu_int8_hip(z)
        dz, again = da.gelu_int8_backward_hip(kept, grad)
        y = da.linear_int8_hip(u, w2, residual=s)
        dx, dw = da.add_rms_norm_backward_hip(s, y, r, weight)
        return s, z, u, dz, again, y, dx, dw

    eager = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for turn in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, captured):
            assert torch.equal(a, b), f"replay {turn}"
        work()
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    """Rows behind 2^32 elements (and bytes): the last ones of a long tensor."""

    device = _device()
    rows, width = 66000, 65536
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=device)
    tail = _randn(40, width, seed=1, dtype=torch.bfloat16)
    x[-40:] = tail
    for group in (None, 128):
        kept = da.quantize_int8_hip(x, group)
        want = da.quantize_int8_hip(tail, group)
        assert torch.equal(kept.values[-40:], want.values) and torch.equal(kept.scales[-40:], want.scales)
        assert not kept.values[:-40].any()
        back = da.dequantize_int8_hip(kept)
        assert torch.equal(back[-40:], da.dequantize_int8_hip(want)) and not back[:-40].any()
        del back
    x = x.view(-1, 16384)
    n = x.shape[0]
    out, total = da.add_rms_norm_hip(x, x)
    assert n * 16384 > 1 << 32 and torch.equal(out[-160:], da.add_rms_norm_hip(x[-160:], x[-160:])[0])
    dx, _ = da.add_rms_norm_backward_hip(total, x, None, None)
    assert torch.equal(dx[-160:], da.add_rms_norm_backward_hip(total[-160:], x[-160:], None, None)[0])
    del out, total, dx
    u, kept = da.gelu_int8_hip(x)
    assert torch.equal(u[-160:], da.gelu_int8_hip(x[-160:])[0])
    dz, _ = da.gelu_int8_backward_hip(kept, x, want_output=False)
    want_dz = da.gelu_int8_backward_hip(da.gelu_int8_hip(x[-160:])[1], x[-160:])[0]
    assert torch.equal(dz[-160:], want_dz)
    del u, kept, dz
    # A linear layer whose output and tokens lie behind 2^32, from both sides.
    wide = x.view(-1, 8192)[:, :64]
    w = da.quantize_int8_hip(_randn(9000, 64, seed=2))
    got = da.linear_int8_hip(wide, w)
    assert got.numel() > 1 << 32
    assert torch.equal(got[-300:], da.linear_int8_hip(wide[-300:], w)) and not got[:1000].any()


def test_launch_on_another_device(monkeypatch) -> None:
    """A launch switches to its tensors' device where another one is current."""

    seen = []

    class Switch:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            seen.append(("enter", self.device))

        def __exit__(self, *_):
            seen.append(("exit", self.device))

    monkeypatch.setattr(int8_ops, "_current_device", lambda: 0)
    monkeypatch.setattr(int8_ops, "_stream", lambda device: ("stream", device.index))
    monkeypatch.setattr(torch.cuda, "device", Switch)
    call = lambda *args: seen.append(args) or 0  # noqa: E731
    int8_ops._launch("test", torch.device("cuda", 0), call, 1, 2)
    assert seen == [(1, 2, ("stream", 0))]
    seen.clear()
    other = torch.device("cuda", 1)
    int8_ops._launch("test", other, call, 3)
    assert seen == [("enter", other), (3, ("stream", 1)), ("exit", other)]


# ---- refusals ------------------------------------------------------------


def test_refusals_on_the_host() -> None:
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    kept = da.QuantizedRows(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4, 1))
    for call in (lambda: da.quantize_int8_hip(x), lambda: da.dequantize_int8_hip(kept), lambda: da.linear_int8_hip(x, kept),
                 lambda: da.linear_int8_hip(kept, kept), lambda: da.add_rms_norm_hip(x), lambda: da.add_rms_norm_int8_hip(x),
                 lambda: da.add_rms_norm_backward_hip(x, x, None, None), lambda: da.gelu_int8_hip(x),
                 lambda: da.gelu_int8_backward_hip(kept._replace(scales=torch.ones(4, 1), group=128), x)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    with pytest.raises(ValueError, match="at least one column"):
        da.quantize_int8_hip(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="float64"):
        da.quantize_int8_hip(torch.zeros(3, 4, dtype=torch.float64))
    for bad in (da.QuantizedRows(kept.values.float(), kept.scales), da.QuantizedRows(kept.values, kept.scales.half()),
                da.QuantizedRows(kept.values, kept.scales[:3]), da.QuantizedRows(kept.values, kept.scales[:, 0]),
                da.QuantizedRows(kept.values, torch.ones(4, 2), 128)):
        with pytest.raises(ValueError):
            da.dequantize_int8_hip(bad)
    with pytest.raises(NotImplementedError):
        da.dequantize_int8_hip(da.QuantizedRows(kept.values, kept.scales, 64))
    with pytest.raises(ValueError, match="activation"):
        da.linear_int8_hip(x, kept, activation="relu")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        da.gelu_int8_hip(torch.zeros(2, 2))


@pytest.mark.gpu
def test_refusals() -> None:
    device = _device()
    x = _randn(4, 8, dtype=torch.bfloat16)
    w = da.quantize_int8_hip(_randn(6, 8))
    b = torch.zeros(6, device=device)
    for call in (lambda: da.linear_int8_hip(x[:, :7], w), lambda: da.linear_int8_hip(x, w, b[:5]),
                 lambda: da.linear_int8_hip(x, w, residual=x), lambda: da.linear_int8_hip(x, w, b.cpu()),
                 lambda: da.linear_int8_hip(x, w, residual=torch.zeros(4, 6, device=device)),
                 lambda: da.linear_int8_hip(x.float(), w), lambda: da.linear_int8_hip(x, w, dtype=torch.float32),
                 lambda: da.linear_int8_hip(da.quantize_int8_hip(x, 128), w),
                 lambda: da.linear_int8_hip(x, da.quantize_int8_hip(_randn(6, 8), 128)),
                 lambda: da.linear_int8_hip(x, w, b.requires_grad_()),
                 lambda: da.add_rms_norm_hip(x, x[:3]), lambda: da.add_rms_norm_hip(x, x.half()),
                 lambda: da.add_rms_norm_hip(x, None, b), lambda: da.add_rms_norm_hip(x, eps=0.0),
                 lambda: da.add_rms_norm_hip(x, eps=float("nan")), lambda: da.add_rms_norm_hip(x.float()),
                 lambda: da.add_rms_norm_int8_hip(x.clone().requires_grad_()),
                 lambda: da.add_rms_norm_backward_hip(x, x[:3], None, None),
                 lambda: da.gelu_int8_hip(x.clone().requires_grad_()),
                 lambda: da.gelu_int8_backward_hip(da.quantize_int8_hip(x), x),
                 lambda: da.gelu_int8_backward_hip(da.quantize_int8_hip(x, 128), x[:3]),
                 lambda: da.quantize_int8_hip(x.double()), lambda: da.dequantize_int8_hip(w, torch.int8)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: da.quantize_int8_hip(torch.zeros(1, 65537, device=device)),
                 lambda: da.quantize_int8_hip(x, 64),
                 lambda: da.add_rms_norm_hip(torch.zeros(1, 16385, device=device, dtype=torch.float16))):
        with pytest.raises(NotImplementedError):
            call()


def test_refusals_of_the_c_abi() -> None:
    """Bad arguments come back as codes before anything is enqueued (no device
    is needed: the pointers are never followed)."""

    if not da.HIP_AVAILABLE:
        pytest.skip("library not built")
    lib = _lib.get()
    p = 4096   # an aligned address that no call reaches
    F32C, F16C = _lib.DA_F32, _lib.DA_F16
    assert lib.da_quantize_int8(p, 2, 8, 8, 7, 0, p, 16, p, None) == -1
    assert lib.da_quantize_int8(p, 2, 8, 8, F16C, 64, p, 16, p, None) == -2
    assert lib.da_quantize_int8(p, 2, 65537, 65537, F16C, 0, p, 65552, p, None) == -2
    assert lib.da_quantize_int8(p, -1, 8, 8, F16C, 0, p, 16, p, None) == -1
    assert lib.da_quantize_int8(p, 2, 0, 8, F16C, 0, p, 16, p, None) == -1
    assert lib.da_quantize_int8(None, 2, 8, 8, F16C, 0, p, 16, p, None) == -1
    assert lib.da_quantize_int8(p + 1, 2, 8, 8, F16C, 0, p, 16, p, None) == -3
    assert lib.da_quantize_int8(p, 2, 8, 7, F16C, 0, p, 16, p, None) == -1
    assert lib.da_quantize_int8(p, 2, 8, 8, F16C, 0, p, 8, p, None) == -3
    assert lib.da_quantize_int8(p, 2, 24, 24, F16C, 0, p, 16, p, None) == -1
    assert lib.da_quantize_int8(p, 2, 8, 8, F16C, 0, p + 8, 16, p, None) == -3
    # Launches of 2^32 threads and more: 16 a group, 64 to 1024 a row.
    assert lib.da_quantize_int8(p, 1 << 28, 8, 8, F16C, 128, p, 16, p, None) == -2
    assert lib.da_quantize_int8(p, 1 << 26, 8, 8, F16C, 0, p, 16, p, None) == -2
    assert lib.da_quantize_int8(p, 1 << 24, 2000, 2000, F16C, 0, p, 2000, p, None) == -2
    assert lib.da_quantize_int8(p, 1 << 22, 20000, 20000, F16C, 0, p, 20000, p, None) == -2
    assert lib.da_dequantize_int8(p, 1 << 27, 256, 256, p, 128, p, 256, F16C, None) == -2
    assert lib.da_gelu_int8(p, 1 << 28, 8, 8, F16C, p, p, 16, p, None) == -2
    assert lib.da_add_rms_norm(p, 8, None, 0, 1 << 26, 8, None, F32C, 1e-6, F16C, None, p, None, 0, None, None) == -2
    assert lib.da_dequantize_int8(p, 2, 8, 16, None, 0, p, 8, F32C, None) == -1
    assert lib.da_dequantize_int8(p, 2, 8, 16, p, 32, p, 8, F32C, None) == -2
    I8C = _lib.DA_I8
    linear = [p, I8C, 16, p, 2, 8, p, 16, p, 6, None, F32C, 0, None, 0, p, F16C, None, 0, None]

    def linear_with(**changes):
        args = list(linear)
        for i, v in changes.items():
            args[int(i[1:])] = v
        return lib.da_linear_int8(*args)

    assert linear_with(_16=F32C) == -1 and linear_with(_12=2) == -1 and linear_with(_9=0) == -2
    assert linear_with(_5=65537, _2=65552, _7=65552) == -2 and linear_with(_2=8) == -3 and linear_with(_7=24) == -3
    assert linear_with(_0=None) == -1 and linear_with(_8=None) == -1 and linear_with(_15=None) == -1
    assert linear_with(_3=None) == -1 and linear_with(_1=F32C) == -1 and linear_with(_7=(1 << 23) + 16) == -2
    assert linear_with(_10=p, _11=9) == -1 and linear_with(_10=p + 2) == -3 and linear_with(_13=p, _14=5) == -1
    assert linear_with(_4=1 << 31) == -2 and linear_with(_4=1 << 18, _9=1 << 17) == -2
    # 16-bit rows that need a workspace: too many columns, or of another type than the output.
    need = lib.da_linear_int8_workspace_bytes(100, 5000, 6, F16C, F16C)
    assert need > 0 and lib.da_linear_int8_workspace_bytes(100, 5000, 6, I8C, F16C) == 0
    wide = {"_1": F16C, "_2": 5000, "_4": 100, "_5": 5000, "_7": 5008}
    assert linear_with(**wide) == -5 and linear_with(**wide, _17=p, _18=need - 1) == -5
    assert linear_with(**wide, _17=p + 8, _18=need) == -3
    assert linear_with(_1=_lib.DA_BF16, _2=8) == -5
    assert lib.da_add_rms_norm(p, 8, None, 0, 2, 8, None, F32C, 0.0, F16C, None, p, None, 0, None, None) == -1
    assert lib.da_add_rms_norm(p, 8, None, 0, 2, 8, None, F32C, 1e-6, F16C, None, None, None, 0, None, None) == -1
    assert lib.da_add_rms_norm(p, 8, p, 8, 2, 8, None, F32C, 1e-6, F16C, None, p, None, 0, None, None) == -1
    assert lib.da_add_rms_norm(p, 8, None, 0, 2, 8, None, F32C, 1e-6, F32C, None, p, None, 0, None, None) == -1
    assert lib.da_add_rms_norm(p, 16385, None, 0, 2, 16385, None, F32C, 1e-6, F16C, None, p, None, 0, None, None) == -2
    need = lib.da_add_rms_norm_backward_workspace_bytes(100, 64)
    assert need > 0
    back = [p, 64, p, 64, None, 0, 100, 64, p, F32C, 1e-6, F16C, p, p, p, need - 1, None]
    assert lib.da_add_rms_norm_backward(*back) == -5
    assert lib.da_add_rms_norm_backward(*back[:14], p + 8, need, None) == -3
    assert lib.da_gelu_int8(p, 2, 8, 8, F32C, p, p, 16, p, None) == -1
    assert lib.da_gelu_int8_backward(p, 2, 8, 16, p, p, 8, F16C, None, None, None) == -1
    # No rows: nothing to do, whatever the pointers are.
    assert lib.da_quantize_int8(None, 0, 8, 8, F16C, 0, None, 16, None, None) == 0
    assert linear_with(_0=None, _3=None, _4=0, _6=None, _15=None) == 0


def test_overlapping_outputs_are_refused_by_the_c_abi() -> None:
    if not da.HIP_AVAILABLE:
        pytest.skip("library not built")
    lib = _lib.get()
    F16C, F32C, I8C = _lib.DA_F16, _lib.DA_F32, _lib.DA_I8
    a, b, c, d = (4096 * (1 + 16 * i) for i in range(4))   # no call reaches them
    # [4, 100] 16-bit rows at a pitch of 104: 824 bytes and 12 behind.
    end = a + 2 * (3 * 104 + 100)

    def norm(x=a, residual=b, total=c, out=d):
        return lib.da_add_rms_norm(x, 104, residual, 104, 4, 100, None, F32C, 1e-6, F16C, total, out, None, 0, None, None)

    for total in (a, a - 798, end - 2, b):
        assert norm(total=total) == -1
    assert norm(out=a) == -1 and norm(out=b) == -1 and norm(out=c) == -1 and norm(out=c + 798) == -1
    assert "overlaps" in _lib.get().da_last_error().decode()

    def back(total=a, grad=b, grad_sum=c, grad_x=d):
        return lib.da_add_rms_norm_backward(total, 100, grad, 100, grad_sum, 100, 4, 100, None, F32C, 1e-6, F16C, grad_x, None,
                                            None, 0, None)

    assert back(grad_x=a) == -1 and back(grad_x=b + 6) == -1 and back(grad_x=c - 6) == -1

    def linear(x=a, weight=b, residual=c, out=d):
        return lib.da_linear_int8(x, I8C, 112, d + 4096, 4, 100, weight, 112, d + 8192, 100, None, F32C, 0, residual, 100, out,
                                  F16C, None, 0, None)

    assert linear(out=a) == -1 and linear(out=b) == -1 and linear(out=c) == -1 and linear(out=c + 798) == -1
    assert lib.da_gelu_int8(a, 4, 100, 104, F16C, end - 2, b, 112, c, None) == -1
    assert lib.da_gelu_int8_backward(a, 4, 100, 112, b, c, 100, F16C, c, None, None) == -1
    assert lib.da_gelu_int8_backward(a, 4, 100, 112, b, c, 100, F16C, d, d, None) == -1


def test_fast_division_is_exact() -> None:
    """The kernels' division by multiplication, as the host sets it up."""

    def setup(d):
        s = (d - 1).bit_length()
        return ((1 << 32) * ((1 << s) - d)) // d + 1, s

    for d in (*range(1, 300), 1000, 4097, 65536, 131072):
        mul, s = setup(d)
        assert mul < 1 << 32
        for n in (0, 1, d - 1, d, d + 1, 7 * d - 1, 7 * d, (1 << 31) - 1, (1 << 31) // d * d - 1, 0x7ffeffff):
            assert (((n * mul) >> 32) + n) >> s == n // d, (n, d)


HEADER = Path(__file__).resolve().parents[1] / "include" / "double_attention_int8.h"


def test_header_declares_what_is_bound() -> None:
    text = HEADER.read_text()
    names = set(re.findall(r"\b(da_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(_lib.INT8_SIGNATURES)
    assert f"#define DA_INT8_GROUP {int8_ops.INT8_GROUP}" in text
    assert f"cols <= {int8_ops.MAX_ROW_COLUMNS}" in text and f"dim <= {int8_ops.MAX_NORM_WIDTH}" in text
