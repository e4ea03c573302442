"""Views whose strides do not matter: dimensions of one element, however far their stride."""

from __future__ import annotations

import pytest
import torch as t

pytestmark = pytest.mark.gpu


def _alone(x, dim, stride):
    """x with that stride in a dimension of size one."""
    strides = list(x.stride())
    assert x.size(dim) == 1
    strides[dim] = stride
    return x.as_strided(x.shape, strides)


@pytest.mark.parametrize("masked", [False, True])
def test_one_key_or_query_at_any_stride(device, masked):
    """A token taken out of a long cache, whose stride to the next is never used, answers bit for
    bit as a copy."""
    from gaussian_splatting.decoder import cross_attention

    gen = t.Generator(device).manual_seed(3)
    randn = lambda *s: t.randn(*s, generator=gen, device=device).bfloat16()  # noqa: E731
    for L, S, H, K in ((1, 1, 2, 1), (1, 40, 2, 1), (5, 1, 2, 1), (1, 1, 1, 1), (100, 1, 1, 1)):
        q, k, v, do = randn(1, L, H, 64), randn(1, S, K, 64), randn(1, S, K, 64), randn(1, L, H, 64)
        mask = t.ones(1, S, device=device, dtype=t.bool) if masked else None

        def run(q, k, v, do):
            leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
            o = cross_attention(*leaves, key_mask=mask)
            return (o, *t.autograd.grad(o, leaves, do))

        want = run(q, k, v, do)
        for far in (1 << 25, 1 << 33, 0):
            moved = [_alone(x, 1, far) if x.size(1) == 1 else x for x in (q, k, v, do)]
            moved = [_alone(x, 2, far) if x.size(2) == 1 else x for x in moved]
            moved = [_alone(x, 0, far) for x in moved]
            got = run(*moved)
            assert all(t.equal(a, b) for a, b in zip(got, want)), (L, S, H, K, far)
