"""The decoder in fp16: trained, and served in 16 and in 8 bits."""

from __future__ import annotations

import pytest
import torch as t

pytestmark = pytest.mark.gpu


def test_fp16_decoder_trains_and_is_served_in_both_widths(device):
    """The attributes of the fp16 and the bf16 model of the same weights differ by bf16's roundings
    (2^-8 of some ten operations in a row, 0.1 at most), the 8-bit answer from the 16-bit one by
    the codes' (2^-4 each, averaged over 64 terms and more: 0.1), and steps lower the loss."""
    from gaussian_splatting.decoder import GaussianDecoder

    def make(dtype):
        t.manual_seed(0)
        return GaussianDecoder(48, width=64, depth=2, heads=4, kv_heads=2, head_dim=32,
                               dtype=dtype).to(device)

    model, wide = make(t.float16), make(t.bfloat16)
    model.load_state_dict({k: v.to(model.state_dict()[k].dtype) for k, v in wide.state_dict().items()})
    gen = t.Generator(device).manual_seed(1)
    tokens = t.randn(2, 40, 48, generator=gen, device=device)
    pos = t.randint(0, 9, (40, 3), generator=gen, device=device)
    query = t.randint(0, 9, (33, 3), generator=gen, device=device)
    with t.no_grad():
        plain = model(tokens.half(), pos, query)
        other = wide(tokens.bfloat16(), pos, query)
        model.serve_in_eight_bits()
        eight = model(tokens.half(), pos, query)
    assert plain.dtype == eight.dtype == t.float32
    assert plain.isfinite().all() and (plain - other).norm() < 0.1 * other.norm()
    assert not t.equal(eight, plain) and (eight - plain).norm() < 0.1 * plain.norm()
    target = t.randn(plain.shape, generator=gen, device=device)
    optimizer = t.optim.SGD(model.parameters(), lr=0.1)
    losses = []
    for _ in range(5):
        loss = (model(tokens.half(), pos, query) - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
        optimizer.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0]
