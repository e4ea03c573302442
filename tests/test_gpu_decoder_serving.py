"""Serving in 8 bits: the 8-bit weights are always those of the weights at the time."""

from __future__ import annotations

import copy

import pytest
import torch as t

pytestmark = pytest.mark.gpu


def _model(device, seed=0):
    from gaussian_splatting.decoder import GaussianDecoder

    t.manual_seed(seed)
    return GaussianDecoder(48, width=64, depth=2, heads=4, kv_heads=2, head_dim=32).to(device)


def _inputs(device):
    gen = t.Generator(device).manual_seed(5)
    tokens = t.randn(2, 7, 48, generator=gen, device=device).bfloat16()
    pos = t.randint(0, 9, (7, 3), generator=gen, device=device)
    query = t.randint(0, 9, (5, 3), generator=gen, device=device)
    return tokens, pos, query


def _fresh_answer(model, inputs):
    """What a model made new with the same weights answers in 8 bits."""
    new = _model(next(model.parameters()).device, seed=99)
    new.load_state_dict({k: v.clone() for k, v in model.state_dict().items()})
    new.serve_in_eight_bits()
    with t.no_grad():
        return new(*inputs)


def _step(model, inputs):
    model(*inputs).square().mean().backward()
    t.optim.SGD(model.parameters(), lr=1.0).step()


def _step_through_data(model, inputs):
    """As a fused optimizer writes: nothing that torch sees."""
    model(*inputs)
    for p in model.parameters():
        p.data.mul_(1.25)


def _in_place(model, inputs):
    with t.no_grad():
        for p in model.parameters():
            p.add_(0.01)


def _load(model, inputs):
    model.load_state_dict(_model(next(model.parameters()).device, seed=3).state_dict())


def _replace(model, inputs):
    for block in model.blocks:
        block.up.weight = t.nn.Parameter(block.up.weight.detach() * 1.5)


def _round_trip(model, inputs):
    device = next(model.parameters()).device
    with t.no_grad():
        for p in model.parameters():
            p.mul_(2)
    model.to("cpu")
    model.to(device)


@pytest.mark.parametrize("change", [_step, _step_through_data, _in_place, _load, _replace, _round_trip])
def test_the_answer_follows_the_weights(device, change):
    model, inputs = _model(device), _inputs(device)
    model.serve_in_eight_bits()
    with t.no_grad():
        before = model(*inputs)
    assert t.equal(before, _fresh_answer(model, inputs))
    change(model, inputs)
    with t.no_grad():
        after = model(*inputs)
        again = model(*inputs)
    assert not t.equal(after, before)
    assert t.equal(after, _fresh_answer(model, inputs)) and t.equal(after, again)


def test_on_and_off(device):
    model, inputs = _model(device), _inputs(device)
    keys = list(model.state_dict())
    with t.no_grad():
        plain = model(*inputs)
    model.serve_in_eight_bits()
    twin = copy.deepcopy(model)
    with t.no_grad():
        eight, twins = model(*inputs), twin(*inputs)
    assert t.equal(eight, twins) and not t.equal(eight, plain)
    assert list(model.state_dict()) == keys
    # with gradients it answers in 16 bits
    assert t.equal(model(*inputs).detach(), plain)
    model.serve_in_eight_bits(False)
    with t.no_grad():
        assert t.equal(model(*inputs), plain)
