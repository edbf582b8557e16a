"""Serving operators at values and sizes off the usual range, against 64-bit forms."""

from __future__ import annotations

import math

import pytest
import torch

import double_attention as da
from test_serving_ops import F32, close, half_step, score_tolerance

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
