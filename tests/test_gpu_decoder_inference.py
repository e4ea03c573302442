"""The decoder's operators without gradients."""

from __future__ import annotations

import pytest
import torch as t

pytestmark = pytest.mark.gpu


def test_positions_that_require_a_gradient_are_data_without_one(device):
    """Learned positions or frequencies: refused where a gradient would be formed, taken as data
    under no_grad and inference_mode."""
    from gaussian_splatting.decoder import axis_frequencies, rotary_axes

    x = t.randn(2, 5, 2, 16, device=device)
    p = t.randn(5, 1, device=device)
    f = axis_frequencies([8]).to(device)
    want = rotary_axes(x, p, f, [8])
    pg, fg = p.clone().requires_grad_(True), f.clone().requires_grad_(True)
    for args in ((pg, f), (p, fg)):
        with pytest.raises(ValueError, match="detach"):
            rotary_axes(x, *args, [8])
    for mode in (t.no_grad, t.inference_mode):
        with mode():
            assert t.equal(rotary_axes(x, pg, fg, [8]), want)
