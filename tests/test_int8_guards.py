"""What the 8-bit operators refuse, and what they do not depend on."""

from __future__ import annotations

import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import double_attention as da
from double_attention import _lib
from test_int8_ops import _device, _randn

F32C, F16C, I8C = _lib.DA_F32, _lib.DA_F16, _lib.DA_I8
REFUSED = -1   # DA_ERR_INVALID_ARGUMENT


def _library():
    if not da.HIP_AVAILABLE:
        pytest.skip("library not built")
    return _lib.get()


def test_import_without_device_support() -> None:
    """A torch that was built for the CPU alone lacks the private device calls:
    the package and its torch backend work there."""

    code = """
import sys
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
sys.path.insert(0, sys.argv[1])
import double_attention as da
config = da.experiment_config("a1", backend="torch", model_dim=32, routing_dim=8, dictionary_size=16)
model = da.DoubleAttentionLM(50, 12, config, 2, feedforward_dim=48, norm="rms")
assert model(torch.zeros(1, 5, dtype=torch.int64))[0].shape == (1, 5, 50)
"""
    package = Path(da.__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code, str(package)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# Buffers of the C calls below, far apart; no refused call follows them.
X, RESIDUAL, WEIGHT, SUM, OUT, VALUES, SCALES, BIAS, SPACE, MORE = (1 << 20 | i << 24 for i in range(1, 11))


def _calls(lib):
    """Each entry point as ``(call(**buffers), buffers written, buffers read)``,
    100 columns of 16-bit rows at a pitch of 104 (inputs) and 6 or 100 rows."""

    def quantize(group):
        def call(x=X, values=VALUES, scales=SCALES):
            return lib.da_quantize_int8(x, 6, 100, 104, F16C, group, values, 112, scales, None)
        return call, {"values": VALUES, "scales": SCALES}, {"x": X}

    def dequantize(out=OUT, values=VALUES, scales=SCALES):
        return lib.da_dequantize_int8(values, 6, 100, 112, scales, 128, out, 104, F16C, None)

    def linear(x=X, x_scales=MORE, weight=WEIGHT, w_scales=SCALES, bias=BIAS, residual=RESIDUAL, out=OUT):
        return lib.da_linear_int8(x, I8C, 112, x_scales, 6, 100, weight, 112, w_scales, 60, bias, F32C, 0, residual, 64, out, F16C,
                                  None, 0, None)

    need = lib.da_linear_int8_workspace_bytes(100, 5000, 60, F16C, F16C)

    def linear16(x=X, weight=WEIGHT, w_scales=SCALES, bias=BIAS, residual=RESIDUAL, out=OUT, workspace=SPACE):
        return lib.da_linear_int8(x, F16C, 5004, None, 100, 5000, weight, 5008, w_scales, 60, bias, F32C, 0, residual, 64, out, F16C,
                                  workspace, need, None)

    def norm(x=X, residual=RESIDUAL, weight=WEIGHT, total=SUM, out=OUT, values=VALUES, scales=SCALES):
        return lib.da_add_rms_norm(x, 104, residual, 104, 6, 100, weight, F32C, 1e-6, F16C, total, out, values, 112, scales, None)

    space = lib.da_add_rms_norm_backward_workspace_bytes(6, 100)

    def norm_backward(total=X, grad=OUT, grad_sum=RESIDUAL, weight=WEIGHT, grad_x=SUM, grad_weight=BIAS, workspace=SPACE):
        return lib.da_add_rms_norm_backward(total, 104, grad, 104, grad_sum, 104, 6, 100, weight, F32C, 1e-6, F16C, grad_x,
                                            grad_weight, workspace, space, None)

    def gelu(z=X, out=OUT, values=VALUES, scales=SCALES):
        return lib.da_gelu_int8(z, 6, 100, 104, F16C, out, values, 112, scales, None)

    def gelu_backward(values=VALUES, scales=SCALES, grad=X, grad_z=OUT, out=SUM):
        return lib.da_gelu_int8_backward(values, 6, 100, 112, scales, grad, 104, F16C, grad_z, out, None)

    return {
        "quantize": quantize(0),
        "quantize in groups": quantize(128),
        "dequantize": (dequantize, {"out": OUT}, {"values": VALUES, "scales": SCALES}),
        "linear": (linear, {"out": OUT}, {"x": X, "x_scales": MORE, "weight": WEIGHT, "w_scales": SCALES, "bias": BIAS,
                                          "residual": RESIDUAL}),
        "linear of 16-bit rows": (linear16, {"out": OUT, "workspace": SPACE},
                                  {"x": X, "weight": WEIGHT, "w_scales": SCALES, "bias": BIAS, "residual": RESIDUAL}),
        "norm": (norm, {"total": SUM, "out": OUT, "values": VALUES, "scales": SCALES},
                 {"x": X, "residual": RESIDUAL, "weight": WEIGHT}),
        "norm backward": (norm_backward, {"grad_x": SUM, "grad_weight": BIAS, "workspace": SPACE},
                          {"total": X, "grad": OUT, "grad_sum": RESIDUAL, "weight": WEIGHT}),
        "gelu": (gelu, {"out": OUT, "values": VALUES, "scales": SCALES}, {"z": X}),
        "gelu backward": (gelu_backward, {"grad_z": OUT, "out": SUM}, {"values": VALUES, "scales": SCALES, "grad": X}),
    }


def test_overlapping_buffers_are_refused_by_the_c_abi() -> None:
    """Every buffer that a call writes, on every other buffer of the call."""

    lib = _library()
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would run on addresses that are none")
    for name, (call, written, read) in _calls(lib).items():
        assert call() != REFUSED, name   # apart: as far as the launch, which fails without a device
        every = {**written, **read}
        for mine in written:
            for other in every:
                if other == mine:
                    continue
                # At its start, and inside its first row (16: the 8-bit rows' alignment).
                assert call(**{mine: every[other]}) == REFUSED, (name, mine, other)
                assert call(**{other: every[mine] + 16}) == REFUSED, (name, mine, other)
                assert "overlaps" in lib.da_last_error().decode()
    # The rest of the last 16 bytes of 8-bit rows is written, too: [6, 100] at a pitch of 112.
    calls = _calls(lib)
    assert calls["quantize"][0](x=VALUES + 6 * 112 - 2) == REFUSED and calls["quantize"][0](x=VALUES + 6 * 112) != REFUSED
    # Without a residual the sum is not written, and without a weight's gradient no workspace.
    assert calls["norm"][0](residual=None, total=X) != REFUSED
    assert calls["norm backward"][0](grad_weight=None, workspace=X) != REFUSED


def test_rows_in_each_others_gaps_are_no_overlap() -> None:
    """Against sets of bytes: only rows of two pitches, both with gaps, go by their ranges."""

    lib = _library()
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would run on addresses that are none")
    rng = random.Random(0)
    seen = set()
    for _ in range(4000):
        rows, cols = rng.randint(1, 5), rng.randint(1, 40)
        ldv = -(-cols // 16) * 16 + 16 * rng.randint(0, 4)
        ldo = (ldv // 2 if rng.random() < 0.5 and ldv // 2 >= cols else cols) + rng.choice((0, 0, rng.randint(0, 40)))
        values = 1 << 20
        out = values + 2 * rng.randint(-rows * ldo - 20, rows * ldv // 2 + 20)
        read = {values + r * ldv + c for r in range(rows) for c in range(cols)}
        wrote = {out + 2 * r * ldo + c for r in range(rows) for c in range(2 * cols)}
        meet = bool(read & wrote)
        if not meet and rows > 1 and ldv > cols and ldo > cols and ldv != 2 * ldo:
            meet = min(read) <= max(wrote) and min(wrote) <= max(read)
        got = lib.da_dequantize_int8(values, rows, cols, ldv, 1 << 28, 0, out, ldo, F16C, None)
        assert (got == REFUSED) == meet, (rows, cols, ldv, ldo, out - values)
        seen.add((meet, max(read) >= min(wrote) and max(wrote) >= min(read)))
    assert seen == {(True, True), (False, True), (False, False)}


@pytest.mark.gpu
def test_rows_in_each_others_gaps() -> None:
    """Rows, their integers and what these stand for as columns of one buffer."""

    lib = _library()
    store = torch.zeros(37, 1024, dtype=torch.uint8, device=_device())
    data = _randn(37, 150, seed=1, dtype=torch.float16)
    store[:, :300] = data.view(torch.uint8)
    scales = torch.zeros(37, 2, device=_device())
    at, stream = store.data_ptr(), torch.cuda.current_stream().cuda_stream
    assert lib.da_quantize_int8(at, 37, 150, 512, F16C, 128, at + 304, 1024, scales.data_ptr(), stream) == 0
    assert lib.da_dequantize_int8(at + 304, 37, 150, 1024, scales.data_ptr(), 128, at + 464, 512, F16C, stream) == 0
    kept = da.quantize_int8_hip(data, 128)
    assert torch.equal(scales, kept.scales) and torch.equal(store[:, 304:454].view(torch.int8), kept.values)
    assert torch.equal(store[:, 464:764].contiguous().view(torch.float16), da.dequantize_int8_hip(kept, torch.float16))
    assert torch.equal(store[:, :300].contiguous().view(torch.float16), data) and not store[:, 764:].any()


def _calls_without_autograd(device):
    """``(call, the tensors that a gradient could be asked of)`` for each operator
    but the norm, which has a backward."""

    x, r, g = (torch.randn(4, 128).bfloat16().to(device) for _ in range(3))
    w, bias = torch.randn(128).to(device), torch.randn(6).to(device)
    kept = lambda scales: da.QuantizedRows(torch.zeros(4, 128, dtype=torch.int8, device=device), scales)  # noqa: E731
    weight = lambda scales: da.QuantizedRows(torch.zeros(6, 128, dtype=torch.int8, device=device), scales)  # noqa: E731
    ones, six = torch.ones(4, 1, device=device), torch.ones(6, 1, device=device)
    return {
        "quantize": (lambda x: da.quantize_int8_hip(x), [x]),
        "dequantize": (lambda scales: da.dequantize_int8_hip(kept(scales)), [ones]),
        "linear": (lambda x, scales, bias, residual: da.linear_int8_hip(x, weight(scales), bias, residual=residual),
                   [x, six, bias, torch.zeros(4, 6, dtype=torch.bfloat16, device=device)]),
        "linear of 8-bit rows": (lambda scales: da.linear_int8_hip(kept(scales), weight(six)), [ones]),
        "norm in 8 bits": (lambda x, r, w: da.add_rms_norm_int8_hip(x, r, w), [x, r, w]),
        "norm backward": (lambda s, g, gs, w: da.add_rms_norm_backward_hip(s, g, gs, w), [x, g, r, w]),
        "gelu": (lambda z: da.gelu_int8_hip(z), [x]),
        "gelu backward": (lambda scales, g: da.gelu_int8_backward_hip(kept(scales)._replace(group=128), g), [ones, g]),
    }


@pytest.mark.gpu
def test_tensors_that_require_grad_are_refused() -> None:
    """No operator drops a gradient that autograd would have recorded."""

    for name, (call, tensors) in _calls_without_autograd(_device()).items():
        call(*tensors)
        for i in range(len(tensors)):
            asked = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate(tensors)]
            with pytest.raises(ValueError, match="no autograd"):
                call(*asked)
            with torch.no_grad():
                call(*asked)


def test_tensors_that_require_grad_are_refused_on_the_host() -> None:
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    scales = torch.ones(4, 1)
    kept = da.QuantizedRows(torch.zeros(4, 128, dtype=torch.int8), scales)
    trained, trained_scales = x.clone().requires_grad_(), scales.clone().requires_grad_()
    for call in (lambda: da.quantize_int8_hip(trained), lambda: da.quantize_int8_hip(trained, 128),
                 lambda: da.dequantize_int8_hip(kept._replace(scales=trained_scales)),
                 lambda: da.add_rms_norm_backward_hip(x, trained, None, None),
                 lambda: da.add_rms_norm_backward_hip(x, x, None, torch.ones(128, requires_grad=True)),
                 lambda: da.gelu_int8_backward_hip(kept._replace(group=128), trained),
                 lambda: da.gelu_int8_backward_hip(kept._replace(scales=trained_scales, group=128), x)):
        with pytest.raises(ValueError, match="no autograd"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="ROCm device"):
            call()


@pytest.mark.gpu
def test_tensors_with_tangents_are_refused() -> None:
    """No operator drops a forward-mode tangent, whether autograd records or not."""

    calls = _calls_without_autograd(_device())
    norm, tensors = calls["norm in 8 bits"]
    calls["norm"] = (da.add_rms_norm_hip, tensors)
    with torch.autograd.forward_ad.dual_level():
        for name, (call, tensors) in calls.items():
            call(*tensors)
            for i in range(len(tensors)):
                dual = [torch.autograd.forward_ad.make_dual(t, t) if i == j else t for j, t in enumerate(tensors)]
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises((ValueError, NotImplementedError), match="forward.mode"):
                        call(*dual)


def test_tensors_with_tangents_are_refused_on_the_host() -> None:
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for call in (lambda: da.quantize_int8_hip(dual), lambda: da.add_rms_norm_int8_hip(x, dual),
                     lambda: da.add_rms_norm_backward_hip(x, dual, None, None)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
