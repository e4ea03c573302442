"""The decoder with nothing to read, or nothing to answer."""

from __future__ import annotations

import pytest
import torch as t

pytestmark = pytest.mark.gpu


def test_a_decoder_without_tokens_or_queries(device):
    """No token: every query answers with what its own embedding gives.  No query, no scene: an
    empty answer, with gradients of 0."""
    from gaussian_splatting.decoder import GaussianDecoder

    t.manual_seed(0)
    model = GaussianDecoder(48, width=64, depth=2, heads=4, kv_heads=2, head_dim=32).to(device)
    tokens = t.randn(2, 7, 48, device=device).bfloat16()
    pos = t.zeros(7, 3, device=device)
    query = t.arange(4, device=device)[:, None].expand(4, 3).contiguous()
    none = model(tokens[:, :0], pos[:0], query)
    padded = model(tokens, pos, query, key_lengths=t.zeros(2, device=device, dtype=t.int32))
    assert none.shape == (2, 4, 59) and t.equal(none, padded)
    for a, p, q in ((tokens, pos, query[:0]), (tokens[:0], pos, query)):
        model.serve_in_eight_bits()
        with t.no_grad():
            assert model(a, p, q).shape == (a.shape[0], q.shape[0], 59)
        out = model(a, p, q)
        assert out.shape == (a.shape[0], q.shape[0], 59)
        model.zero_grad()
        out.sum().backward()
        assert (model.query.grad == 0).all()
