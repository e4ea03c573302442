"""A second differentiation of the decoder's operators: refused wherever a first gradient depends
on an input that requires one, also where the gradient that came in is a constant."""

from __future__ import annotations

import pytest
import torch as t

pytestmark = pytest.mark.gpu


def _parts(device):
    import gaussian_splatting.decoder as ops

    gen = t.Generator(device).manual_seed(0)
    randn = lambda *s: t.randn(*s, generator=gen, device=device).bfloat16()  # noqa: E731
    pos = t.arange(5, device=device)[:, None]
    inv = ops.axis_frequencies([8]).to(device)
    x, k, v, w = randn(2, 5, 2, 16), randn(2, 9, 2, 16), randn(2, 9, 2, 16), randn(16)
    return ops, pos, inv, x, k, v, w


def _gradient_penalty(call, leaves, of):
    """backward of |d sum(call) / d of|^2 and a term of its own."""
    y = call(*leaves)
    g, = t.autograd.grad(y.float().sum(), of, create_graph=True)
    (g.float().square().sum() + sum(x.float().sum() for x in leaves)).backward()


def test_a_constant_incoming_gradient_is_refused_too(device):
    """sum(o)'s gradient is a constant, its own derivative is not 0: dropping it would leave the
    penalty out of the step without a word."""
    ops, _, _, x, k, v, w = _parts(device)
    calls = [
        (lambda a, b, c: ops.cross_attention(a, b, c), (x, k, v), 0),
        (lambda a, b, c: ops.cross_attention(a, b, c), (x, k, v), 2),
        (lambda a, b: ops.rms_norm_residual(a, None, b)[0], (x, w), 0),
        (lambda a, b: ops.rms_norm_residual(a, None, b)[0], (x, w), 1),
        (lambda a, b: ops.rms_norm_residual(a, a.detach(), b)[0], (x, w), 0),
    ]
    for call, inputs, of in calls:
        leaves = [z.detach().clone().requires_grad_(True) for z in inputs]
        with pytest.raises(RuntimeError, match="once"):
            _gradient_penalty(call, leaves, leaves[of])


def test_gradients_that_are_constant_are_not_refused(device):
    """rotary_axes is linear in x, o in v and y in the weight: with only that input wanting a
    gradient, the penalty's derivative is 0 and the other term's 1 is what arrives."""
    ops, pos, inv, x, k, v, w = _parts(device)
    calls = [(lambda z: ops.rotary_axes(z, pos, inv, [8]), x),
             (lambda z: ops.cross_attention(x, k, z), v),
             (lambda z: ops.rms_norm_residual(x, x, z)[0], w)]
    for call, z in calls:
        leaf = z.detach().clone().requires_grad_(True)
        _gradient_penalty(call, [leaf], leaf)
        assert (leaf.grad == 1).all()


def test_h_alone_passes_its_gradient_through_twice(device):
    """h = x + residual: the gradient through h alone is the one that came in."""
    ops, _, _, x, _, _, w = _parts(device)
    leaf = x.detach().clone().requires_grad_(True)
    _, h = ops.rms_norm_residual(leaf, x, w)
    g, = t.autograd.grad(h.float().square().sum(), leaf, create_graph=True)
    g.float().sum().backward()
    assert (leaf.grad == 2).all()
