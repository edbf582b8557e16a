"""The blocks and the language model on the 8-bit operators.

* ``norm="rms"``: root-mean-square norms, with the residual's addition in front
  of the second one, in inference and training;
* ``quantize_feedforward()``: the feed-forward on 8-bit integers in inference;
* ``activation_checkpoint="int8"``: the feed-forward's saved activations in
  8 bits, and their use in the backward pass.
"""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import double_attention as da
from test_int8_ops import HALF, _device, _randn, groups_of


def _block(dtype, *, preset="a1", feedforward_dim=320, **options):
    torch.manual_seed(0)
    config = da.experiment_config(preset, backend="hip", model_dim=128, **options.pop("config", {}))
    block = da.DoubleAttentionBlock(config, feedforward_dim=feedforward_dim, **options)
    bank = da.SharedDictionaryBank(config.routing_dim, config.dictionary_size, untied=config.untied_dictionary)
    with torch.no_grad():
        for p in block.parameters():
            if p.ndim == 1 and p.numel() == 128:
                p.add_(0.1 * torch.randn(p.shape))
    return block.to(_device(), dtype), bank.to(_device(), dtype)


def rel(got, expected):
    got, expected = got.double(), expected.double()
    return ((got - expected).norm() / expected.norm()).item()


def feedforward64(block, h):
    """W2 GELU(W1 h + b1) + b2 in 64 bits."""

    first, second = block.feedforward[0], block.feedforward[2]
    z = F.linear(h.double(), first.weight.double(), first.bias.double())
    return F.linear(0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5)), second.weight.double(), second.bias.double())


def test_options_on_the_host() -> None:
    config = da.experiment_config("a1", backend="torch", model_dim=32, routing_dim=8, dictionary_size=16)
    with pytest.raises(ValueError, match="norm"):
        da.DoubleAttentionBlock(config, norm="batch")
    with pytest.raises(ValueError, match="activation_checkpoint"):
        da.DoubleAttentionBlock(config, activation_checkpoint="fp8")
    plain = da.DoubleAttentionLM(50, 12, config, 2, feedforward_dim=48)
    rms = da.DoubleAttentionLM(50, 12, config, 2, feedforward_dim=48, norm="rms", activation_checkpoint="int8")
    names = {n for n in plain.state_dict() if not n.endswith("norm.bias")}
    assert set(rms.state_dict()) == names
    assert all(isinstance(m, nn.RMSNorm) for m in (rms.final_norm, rms.stack.blocks[1].attention_norm))
    # Without the kernels the model runs as it is, the options' gradients too.
    ids = torch.randint(0, 50, (3, 12), generator=torch.Generator().manual_seed(0))
    logits, loss = rms(ids, ids)
    loss.backward()
    assert logits.shape == (3, 12, 50) and rms.stack.blocks[0].feedforward_norm.weight.grad.abs().sum() > 0
    with pytest.raises(ValueError, match="ROCm device"):
        rms.quantize_feedforward()
    rms.quantize_feedforward(False)


def test_q_dictionary_feedforward_is_refused() -> None:
    config = da.experiment_config("a1-d1536-qffn", backend="torch")
    with pytest.raises(ValueError, match="Q-dictionary"):
        da.DoubleAttentionBlock(config, feedforward_dim=config.dictionary_size, activation_checkpoint="int8")
    block = da.DoubleAttentionBlock(config, feedforward_dim=config.dictionary_size)
    with pytest.raises(NotImplementedError):
        block.quantize_feedforward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("output_projection", [True, False])
def test_rms_block_is_its_stages(dtype, output_projection) -> None:
    """The block against its attention and 64-bit norms and feed-forward: each
    stage rounds to 16 bits (norm, GELU, output, sums: at most 6 half steps
    of the largest term)."""

    block, bank = _block(dtype, norm="rms", config={"output_projection": output_projection})
    x = _randn(3, 17, 128, seed=1, dtype=dtype)

    def norm64(norm, t):
        t = t.double()
        return t * (t.square().mean(-1, keepdim=True) + norm.eps).rsqrt() * norm.weight.double()

    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            got = block(x, bank)
        with torch.no_grad():
            n1 = norm64(block.attention_norm, x).to(dtype)
            s = x.double() + block.attention(n1, bank=bank).double()
            y = s + feedforward64(block, norm64(block.feedforward_norm, s.to(dtype)))
        assert rel(got, y) < 6 * torch.finfo(dtype).eps / 2
    assert isinstance(block.feedforward_norm, nn.RMSNorm)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_rms_block_gradients(dtype) -> None:
    """Against the torch composition in fp32 on the same weights."""

    block, bank = _block(dtype, norm="rms")
    x = _randn(2, 40, 128, seed=1, dtype=dtype)
    g = _randn(2, 40, 128, seed=2, dtype=dtype)

    def grads(block, bank, x, g):
        x = x.clone().requires_grad_()
        block.zero_grad(set_to_none=True)
        bank.zero_grad(set_to_none=True)
        block(x, bank).backward(g)
        return {"x": x.grad, **{n: p.grad for n, p in block.named_parameters() if p.grad is not None}}

    got = grads(block, bank, x, g)
    reference = da.DoubleAttentionBlock(da.experiment_config("a1", backend="torch", model_dim=128), feedforward_dim=320,
                                        norm="rms").to(_device())
    reference.load_state_dict({n: p.float() for n, p in block.state_dict().items()})
    want = grads(reference, copy.deepcopy(bank).float(), x.float(), g.float())
    assert set(got) == set(want)
    for name in want:
        if want[name].numel() > 4:   # beta and the temperature are sums that cancel
            assert rel(got[name], want[name]) < 3e-2, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_quantized_feedforward(norm, dtype) -> None:
    block, bank = _block(dtype, norm=norm)
    x = _randn(2, 33, 128, seed=1, dtype=dtype)
    with torch.no_grad():
        full = block(x, bank)
        block.quantize_feedforward()
        got = block(x, bank)
        # The same calls by hand.
        attention, norm2 = block.attention, block.feedforward_norm
        n1 = block.attention_norm
        if norm == "rms":
            h = da.add_rms_norm_hip(x, None, n1.weight, n1.eps)[0]
        else:
            h = da.hip_ops.layer_norm_hip(x, n1.weight, n1.bias, n1.eps)
        s = attention._hip_call(h, bank, None, dtype, residual=x, want_routed=False).output
        first, second = block.feedforward[0], block.feedforward[2]
        w1, w2 = da.quantize_int8_hip(first.weight), da.quantize_int8_hip(second.weight)
        if norm == "rms":
            h = da.add_rms_norm_int8_hip(s, None, norm2.weight, norm2.eps)[0]
        else:
            h = da.hip_ops.layer_norm_hip(s, norm2.weight, norm2.bias, norm2.eps)
        u = da.linear_int8_hip(h, w1, first.bias, activation="gelu", dtype=dtype)
        assert torch.equal(got, da.linear_int8_hip(u, w2, second.bias, residual=s))
        # A value is off by at most half a step of amax / 127; over 128 or 320
        # normal values (amax about 3 deviations, a few channels larger) that is
        # about 1% of a deviation, in each of four operands.
        assert rel(got - s, full - s) < 4e-2
        # Autograd keeps the full weights; dropping the 8-bit ones, too.
    y = block(x.clone().requires_grad_(), bank)
    assert rel(y, full) < 2 * torch.finfo(dtype).eps
    block.quantize_feedforward(False)
    with torch.no_grad():
        assert torch.equal(block(x, bank), full)
        block.quantize_feedforward()
        second.weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="quantize_feedforward"):
            block(x, bank)
        block.quantize_feedforward()
        block(x, bank)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 2])
def test_quantized_feedforward_of_replaced_weights(which) -> None:
    """A parameter put in a weight's place has the weight's version, not its values."""

    block, bank = _block(torch.bfloat16)
    x = _randn(2, 5, 128, seed=1, dtype=torch.bfloat16)
    with torch.no_grad():
        block.quantize_feedforward()
        block(x, bank)
        linear = block.feedforward[which]
        kept = linear.weight
        linear.weight = nn.Parameter(-kept)
        while linear.weight._version < kept._version:
            linear.weight.mul_(1.0)
        assert linear.weight._version == kept._version
        with pytest.raises(RuntimeError, match="quantize_feedforward"):
            block(x, bank)
        linear.weight = kept
        block(x, bank)


@pytest.mark.gpu
def test_quantized_feedforward_without_output_projection() -> None:
    """The block that does not run as one fused forward takes the 8-bit weights, too."""

    block, bank = _block(torch.bfloat16, norm="rms", config={"output_projection": False})
    x = _randn(2, 33, 128, seed=1, dtype=torch.bfloat16)
    with torch.inference_mode():
        full = block(x, bank)
        block.quantize_feedforward()
        got = block(x, bank)
        assert not torch.equal(got, full) and rel(got, full) < 4e-2
        # The residual's addition, the norm and its integers in one call.
        n1, n2 = block.attention_norm, block.feedforward_norm
        attended = block.attention(da.add_rms_norm_hip(x, None, n1.weight, n1.eps)[0], bank=bank)
        kept, s = da.add_rms_norm_int8_hip(attended, x, n2.weight, n2.eps)
        first, second = block.feedforward[0], block.feedforward[2]
        w1, w2 = da.quantize_int8_hip(first.weight), da.quantize_int8_hip(second.weight)
        u = da.linear_int8_hip(kept, w1, first.bias, activation="gelu", dtype=torch.bfloat16)
        assert torch.equal(got, da.linear_int8_hip(u, w2, second.bias, residual=s))
    # Autograd takes the full weights there, too.
    y = block(x, bank)
    assert y.requires_grad and rel(y, full) < 2 * torch.finfo(torch.bfloat16).eps


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_quantized_language_model_and_its_graph(norm) -> None:
    device = _device()
    torch.manual_seed(0)
    config = da.experiment_config("qk2-s2", untied_dictionary=False, backend="hip")
    model = da.DoubleAttentionLM(300, 40, config, 2, feedforward_dim=1536, norm=norm).to(device, torch.bfloat16).eval()
    ids = torch.randint(0, 300, (5, 33), generator=torch.Generator().manual_seed(1)).to(device)
    one = ids[:1, :1]
    with torch.inference_mode():
        full, full_one = model(ids)[0], model(one)[0]
        model.quantize_feedforward()
        got, got_one = model(ids)[0], model(one)[0]
    # The residual stream carries most of the logits: the feed-forwards' 4% of them.
    assert rel(got, full) < 4e-2 and rel(got_one, full_one) < 4e-2
    graphed = da.GraphedForward(lambda t: model(t)[0], ids)
    other = torch.randint(0, 300, (5, 33), generator=torch.Generator().manual_seed(2)).to(device)
    for turn in range(3):
        for t in (ids, other):
            replayed = graphed(t).clone()
            with torch.inference_mode():
                assert torch.equal(replayed, model(t)[0]), turn
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_activation_checkpoint(norm, dtype) -> None:
    """The forward's values are those of the 16-bit function; the gradients are
    the formula's on the rows as they were kept."""

    block, bank = _block(dtype, norm=norm, activation_checkpoint="int8")
    plain = copy.deepcopy(block)
    plain.activation_checkpoint = None
    x = _randn(3, 50, 128, seed=1, dtype=dtype)
    g = _randn(3, 50, 128, seed=2, dtype=dtype)

    def step(block):
        leaf = x.clone().requires_grad_()
        block.zero_grad(set_to_none=True)
        y = block(leaf, bank)
        y.backward(g)
        return y.detach(), leaf.grad, {n: p.grad for n, p in block.named_parameters() if p.grad is not None}

    y, dx, got = step(block)
    y0, dx0, want = step(plain)
    # GELU is the same function in two formulas, one rounding apart.
    assert rel(y, y0) < torch.finfo(dtype).eps and set(got) == set(want)
    # A kept value is off by at most half a step, amax / 254 of its group: 0.6%
    # of a deviation for normal values, more where a channel is large.
    assert rel(dx, dx0) < 2e-2
    for name in want:
        if want[name].numel() > 4:
            assert rel(got[name], want[name]) < 2e-2, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(1, 128), (3, 7, 128), (300, 128), (0, 128)])
def test_feedforward_function_gradients(shape, dtype) -> None:
    """Each gradient of the feed-forward against its formula in 64 bits on what
    the kept rows stand for."""

    from double_attention.modules import _HipFeedForwardInt8Function

    device = _device()
    torch.manual_seed(1)
    w1, b1 = (torch.randn(320, 128) * 128 ** -0.5), 0.1 * torch.randn(320)
    w2, b2 = (torch.randn(128, 320) * 320 ** -0.5), 0.1 * torch.randn(128)
    params = [t.to(device, dtype).requires_grad_() for t in (w1, b1, w2, b2)]
    x, h, g = (_randn(*shape, seed=s, dtype=dtype) for s in (1, 2, 3))
    x, h = x.requires_grad_(), h.requires_grad_()
    if not x.numel():
        # As the 16-bit function: the linear layer in front refuses no tokens.
        with pytest.raises(ValueError, match="linear"):
            _HipFeedForwardInt8Function.apply(x, h, *params)
        return
    y = _HipFeedForwardInt8Function.apply(x, h, *params)
    grads = torch.autograd.grad(y, (x, h, *params), g)
    assert torch.equal(grads[0], g)
    assert all(t.shape == p.shape and t.dtype == p.dtype for t, p in zip(grads, (x, h, *params)))
    def stands(t):
        kept = da.quantize_int8_hip(t, 128)
        return (groups_of(kept.values.double(), 128) * kept.scales.double().unsqueeze(-1)).flatten(-2)[..., : t.shape[-1]]

    W1, B1, W2, _ = (p.detach().double() for p in params)
    z = da.hip_ops.linear_hip(h.detach(), params[0].detach(), params[1].detach())
    zt = stands(z).flatten(0, -2)
    below = 0.5 * (1 + torch.erf(zt * 0.5 ** 0.5))
    slope = below + zt * torch.exp(-0.5 * zt * zt) * (2 * torch.pi) ** -0.5
    dy = g.double().flatten(0, -2)
    dz = dy @ W2 * slope
    want = (dz @ W1, dz.t() @ stands(h.detach()).flatten(0, -2), dz.sum(0), dy.t() @ (zt * below), dy.sum(0))
    # dU, dZ, u and h round to 16 bits on the way, and so do the results:
    # in the 2-norm, at most five half steps.
    for name, got, expected in zip(("h", "w1", "b1", "w2", "b2"), grads[1:], want):
        assert rel(got.reshape(expected.shape), expected) < 5 * torch.finfo(dtype).eps / 2, name


@pytest.mark.gpu
def test_activation_checkpoint_saves_memory() -> None:
    """What a feed-forward of 512 -> 1536 holds between forward and backward."""

    from double_attention.modules import _HipFeedForwardFunction, _HipFeedForwardInt8Function

    device = _device()
    params = [torch.randn(*s, device=device).bfloat16().requires_grad_() for s in ((1536, 512), (1536,), (512, 1536), (512,))]
    held = []
    for function in (_HipFeedForwardFunction, _HipFeedForwardInt8Function):
        x = torch.randn(8192, 512, device=device).bfloat16().requires_grad_()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = function.apply(x, x * 1.0, *params)
        held.append((torch.cuda.memory_allocated() - before - y.numel() * 2) / x.numel())
        y.backward(y.detach())
        del y, x
    # Bytes for each feature of x: h, z and u in 16 bits; h and z in 8 with a
    # scale for each 128.
    assert held[0] >= 2 + 6 + 6 and held[1] <= 4 * (1 + 4 / 128) + 0.1


@pytest.mark.gpu
def test_training_step_of_a_checkpointed_language_model() -> None:
    device = _device()
    torch.manual_seed(0)
    config = da.experiment_config("qk2-s2", untied_dictionary=False, backend="hip")
    model = da.DoubleAttentionLM(300, 40, config, 2, feedforward_dim=1536, norm="rms", activation_checkpoint="int8")
    model = model.to(device, torch.bfloat16)
    ids = torch.randint(0, 300, (4, 40), generator=torch.Generator().manual_seed(1)).to(device)
    # The next token: a token's own logit under the tied embedding is so large
    # that learning the token itself has no gradient at all.
    targets = ids.roll(-1, dims=1)
    _, loss = model(ids, targets)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    assert all(torch.isfinite(t).all() for t in got.values())
    for block in model.stack.blocks:
        block.activation_checkpoint = None
    model.zero_grad(set_to_none=True)
    model(ids, targets)[1].backward()
    for name, p in model.named_parameters():
        if p.numel() > 4:
            assert rel(got[name], p.grad) < 4e-2, name   # two layers of the 2e-2 of one
