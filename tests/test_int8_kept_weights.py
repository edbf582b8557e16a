"""The feed-forward's 8-bit weights when the block around them is copied, saved,
changed or captured."""

from __future__ import annotations

import copy
import io

import pytest
import torch

import double_attention as da
from double_attention import int8_ops
from test_int8_modules import _block
from test_int8_ops import _randn


def _quantized(x, group=None):
    """``quantize_int8_hip`` of weights, on the host."""

    assert group is None
    scales = x.detach().float().abs().amax(-1, keepdim=True) / 127
    return da.QuantizedRows(torch.round(x.detach().float() / scales).to(torch.int8), scales)


def _host_block(monkeypatch, **options):
    """A block on the host, its weights written in place as by a checkpoint."""

    monkeypatch.setattr(int8_ops, "quantize_int8_hip", _quantized)
    config = da.experiment_config("a1", backend="torch", model_dim=32, routing_dim=8, dictionary_size=16)
    torch.manual_seed(0)
    block = da.DoubleAttentionBlock(config, feedforward_dim=48, **options)
    block.load_state_dict({n: p + 0.01 for n, p in block.state_dict().items()})
    return block


def _copies(block):
    file = io.BytesIO()
    torch.save(block, file)
    file.seek(0)
    return copy.deepcopy(block), copy.copy(block), torch.load(file, weights_only=False), copy.deepcopy(copy.deepcopy(block))


def test_copies_of_a_quantized_block(monkeypatch) -> None:
    """A copy has the 8-bit weights of its own parameters, and sees these change."""

    block = _host_block(monkeypatch)
    block.quantize_feedforward()
    want = block._int8_weights()
    for other in _copies(block):
        for got, expected in zip(other._int8_weights(), want):
            assert torch.equal(got.values, expected.values) and torch.equal(got.scales, expected.scales)
    deep = copy.deepcopy(block)
    assert deep._int8_weights()[0].values.data_ptr() != want[0].values.data_ptr()
    with torch.no_grad():
        deep.feedforward[2].weight.mul_(2.0)
    with pytest.raises(RuntimeError, match="quantize_feedforward"):
        deep._int8_weights()
    assert block._int8_weights() is want
    deep.quantize_feedforward()
    assert torch.equal(deep._int8_weights()[1].scales, 2 * want[1].scales)


def test_copies_of_a_block_whose_weights_changed(monkeypatch) -> None:
    """They know no more about their 8-bit weights than the block itself."""

    block = _host_block(monkeypatch)
    block.quantize_feedforward()
    with torch.no_grad():
        block.feedforward[0].weight.add_(1.0)
    for other in (block, *_copies(block)):
        with pytest.raises(RuntimeError, match="quantize_feedforward"):
            other._int8_weights()


def test_inference_tensors_as_weights(monkeypatch) -> None:
    """Nothing tells when they are written: no 8-bit weights are kept of them."""

    with torch.inference_mode():
        block = _host_block(monkeypatch)
        with pytest.raises(ValueError, match="inference_mode"):
            block.quantize_feedforward()
        assert block._int8_weights() is None
    # Copies made there are such tensors, too, whatever the block's own are.
    block = _host_block(monkeypatch)
    with torch.inference_mode():
        block.quantize_feedforward()
        assert block._int8_weights() is not None
        other = copy.deepcopy(block)
        assert other.feedforward[0].weight.is_inference()
        with pytest.raises(RuntimeError, match="quantize_feedforward"):
            other._int8_weights()


def _saved_before(block):
    """The block as an older version saved it whole."""

    state = block.__dict__.copy()
    state.pop("activation_checkpoint")
    state.pop("_int8_feedforward", None)
    other = block.__class__.__new__(block.__class__)
    other.__setstate__(state)
    return other


def test_block_that_was_saved_without_the_attributes(monkeypatch) -> None:
    block = _host_block(monkeypatch)
    bank = da.SharedDictionaryBank(8, 16)
    x = torch.randn(2, 5, 32, generator=torch.Generator().manual_seed(1))
    old = _saved_before(block)
    assert torch.equal(old(x, bank), block(x, bank))
    old.quantize_feedforward()
    assert old._int8_weights() is not None and block._int8_weights() is None


@pytest.mark.gpu
def test_old_block_on_the_kernels() -> None:
    block, bank = _block(torch.bfloat16)
    old = _saved_before(block)
    x = _randn(2, 33, 128, seed=1, dtype=torch.bfloat16)
    with torch.no_grad():
        assert torch.equal(old(x, bank), block(x, bank))
    assert torch.equal(old(x, bank), block(x, bank))


@pytest.mark.gpu
def test_forward_of_a_copied_quantized_block() -> None:
    block, bank = _block(torch.bfloat16, norm="rms")
    x = _randn(2, 33, 128, seed=1, dtype=torch.bfloat16)
    block.load_state_dict({n: p * 1.0 for n, p in block.state_dict().items()})
    with torch.no_grad():
        block.quantize_feedforward()
        want = block(x, bank)
        for other in _copies(block):
            assert torch.equal(other(x, bank), want)


def test_weights_quantized_again_keep_their_memory(monkeypatch) -> None:
    """A captured graph reads the 8-bit weights where they were."""

    block = _host_block(monkeypatch)
    with torch.inference_mode():
        block.quantize_feedforward()
    kept = block._int8_weights()
    places = [t.data_ptr() for rows in kept for t in rows[:2]]
    with torch.no_grad():
        for i in (0, 2):
            block.feedforward[i].weight.mul_(-2.0)
    with pytest.raises(RuntimeError, match="quantize_feedforward"):
        block._int8_weights()
    block.quantize_feedforward()
    again = block._int8_weights()
    assert [t.data_ptr() for rows in again for t in rows[:2]] == places
    for i, rows in zip((0, 2), again):
        want = _quantized(block.feedforward[i].weight)
        assert torch.equal(rows.values, want.values) and torch.equal(rows.scales, want.scales)
    # Other parameters in the weights' place, and weights of another shape.
    block.feedforward[0].weight = torch.nn.Parameter(torch.randn(48, 32))
    block.quantize_feedforward()
    assert block._int8_weights()[0].values.data_ptr() == places[0]
    block.feedforward[0] = torch.nn.Linear(32, 40)
    block.feedforward[2] = torch.nn.Linear(40, 32)
    block.quantize_feedforward()
    assert block._int8_weights()[0].values.shape == (40, 32)


def test_uses_of_8_bit_weights_are_collected(monkeypatch) -> None:
    from double_attention.modules import int8_weights_used

    first, second = _host_block(monkeypatch), _host_block(monkeypatch)
    first.quantize_feedforward()
    second.quantize_feedforward()
    with int8_weights_used() as outer:
        first._int8_weights()
        with int8_weights_used() as inner:
            second._int8_weights()
            second._int8_weights()
    first._int8_weights()
    assert inner == [second._int8_feedforward] and outer == [first._int8_feedforward, second._int8_feedforward]


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_captured_forward_and_changed_weights(norm) -> None:
    """A replay has the weights as they were quantized last, and refuses where
    they changed since; dropped 8-bit weights stay with the graph."""

    block, bank = _block(torch.bfloat16, norm=norm)
    x = _randn(2, 33, 128, seed=1, dtype=torch.bfloat16)
    block.quantize_feedforward()
    graphed = da.GraphedForward(lambda t: block(t, bank), x)

    def eager():
        with torch.no_grad():
            return block(x, bank)

    before = eager()
    assert torch.equal(graphed(x), before)
    for turn in range(3):
        with torch.no_grad():
            block.feedforward[0].weight.mul_(-1.5)
            block.feedforward[2].weight.add_(0.1 * torch.randn_like(block.feedforward[2].weight))
        with pytest.raises(RuntimeError, match="quantize_feedforward"):
            graphed(x)
        block.quantize_feedforward()
        want = eager()
        assert not torch.equal(want, before), turn
        assert torch.equal(graphed(x), want), turn
        torch.cuda.synchronize()
        before = want
    block.quantize_feedforward(False)
    fill = [torch.full((1 << 16,), 85, dtype=torch.int8, device=x.device) for _ in range(64)]
    assert torch.equal(graphed(x), before) and not torch.equal(eager(), before)
    torch.cuda.synchronize()
    del fill
