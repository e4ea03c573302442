"""A decoder that reads the tokens of posed views and answers with Gaussians, which the
rasterizer renders and trains through: the decoder operators as they are used together.

Every query is anchored at a pixel of one view.  A block adds to the residual stream what the
queries read from the views' tokens (norm, projection, rotary positions of query and token,
cross attention) and what a two-layer network makes of it; the head gives each query the 59
attributes of a Gaussian on its pixel's ray.
"""

from __future__ import annotations

import torch as t
from torch import nn

from gaussian_splatting.decoder.attention import cross_attention
from gaussian_splatting.decoder.norm import rms_norm_residual, rms_norm_residual_fp8
from gaussian_splatting.decoder.rotary import axis_frequencies, rotary_axes
from gaussian_splatting.scene.gaussian import gaussian

ATTRIBUTES = 59  # offset on the pixel 2, depth 1, q 4, log-scales 3, opacity logit 1, A 3, k_j 45


def patch_tokens(image: t.Tensor, patch: int = 16) -> tuple[t.Tensor, t.Tensor]:
    """((S, 3 patch^2) pixels, (S, 3) positions (view 0, row, column)) of an (H, W, 3) image;
    the last row and column of patches are filled with zeros."""
    H, W, _ = image.shape
    rows, cols = -(-H // patch), -(-W // patch)
    full = image.new_zeros(rows * patch, cols * patch, 3)
    full[:H, :W] = image
    tokens = full.reshape(rows, patch, cols, patch, 3).permute(0, 2, 1, 3, 4)
    r = t.arange(rows, device=image.device).repeat_interleave(cols)
    c = t.arange(cols, device=image.device).repeat(rows)
    return (tokens.reshape(rows * cols, patch * patch * 3),
            t.stack((t.zeros_like(r), r, c), -1))


class DecoderBlock(nn.Module):
    def __init__(self, width: int, token_width: int, heads: int, kv_heads: int, head_dim: int,
                 dtype: t.dtype) -> None:
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        make = lambda a, b: nn.Linear(a, b, bias=False, dtype=dtype)  # noqa: E731
        self.norm_attention = nn.Parameter(t.ones(width, dtype=dtype))
        self.norm_network = nn.Parameter(t.ones(width, dtype=dtype))
        self.to_q = make(width, heads * head_dim)
        self.to_kv = make(token_width, 2 * kv_heads * head_dim)
        self.out = make(heads * head_dim, width)
        self.up = make(width, 4 * width)
        self.down = make(4 * width, width)
        self._eight_bit = None

    def eight_bit_weight(self) -> tuple[t.Tensor, t.Tensor]:
        """(codes, a scale per output) of ``up``'s weight, formed when first asked for and again
        whenever the weight has changed: in place (its version says so), replaced, moved or
        converted, or, with whatever wrote to it, after a forward with gradients."""
        w = self.up.weight
        version = None if w.is_inference() else w._version
        if self._eight_bit is None or self._eight_bit[0] is not w or self._eight_bit[1] != version:
            values = w.detach().float()
            scale = values.abs().amax(1).clamp(min=1e-12) / 448.0
            codes = (values / scale[:, None]).to(t.float8_e4m3fn)
            self._eight_bit = (w, version, codes, scale)
        return self._eight_bit[2:]

    def forget_eight_bit_weight(self) -> None:
        self._eight_bit = None

    def _apply(self, *args, **kwargs):  # to(), half(), ...
        self.forget_eight_bit_weight()
        return super()._apply(*args, **kwargs)

    def forward(self, x, residual, tokens, query_pos, token_pos, inv_freq, sections, key_lengths,
                key_mask, eight_bit=False):
        """(x, residual) after the block: x is still to be added to the residual stream."""
        B, L, _ = x.shape
        y, residual = rms_norm_residual(x, residual, self.norm_attention)
        q = self.to_q(y).view(B, L, self.heads, self.head_dim)
        kv = self.to_kv(tokens).view(B, tokens.shape[1], 2, self.kv_heads, self.head_dim)
        q = rotary_axes(q, query_pos, inv_freq, sections)
        k = rotary_axes(kv[:, :, 0], token_pos, inv_freq, sections)
        o = cross_attention(q, k, kv[:, :, 1], key_lengths=key_lengths, key_mask=key_mask)
        o = self.out(o.flatten(-2))
        if not eight_bit:
            y, residual = rms_norm_residual(o, residual, self.norm_network)
            return self.down(nn.functional.gelu(self.up(y))), residual
        y8, scale, residual = rms_norm_residual_fp8(o, residual, self.norm_network)
        weight, weight_scale = self.eight_bit_weight()
        # the library's product with a scale per row answers in bf16 only, whose 2^-9 is small
        # beside the codes' 2^-4
        h = t._scaled_mm(y8.flatten(0, -2), weight.t(), scale_a=scale.reshape(-1, 1),
                         scale_b=weight_scale.reshape(1, -1), out_dtype=t.bfloat16).to(o.dtype)
        return self.down(nn.functional.gelu(h.view(B, L, h.shape[1]))), residual


class GaussianDecoder(nn.Module):
    """Gaussians from the tokens of posed views.

    Args:
        token_width: width of the views' tokens
        width, depth, heads, kv_heads, head_dim: of the decoder (head_dim a multiple of 8
            up to 128)
        dtype: of the weights and activations, torch.bfloat16 or torch.float16
    """

    def __init__(self, token_width: int, width: int = 256, depth: int = 2, heads: int = 8,
                 kv_heads: int = 2, head_dim: int = 64, dtype: t.dtype = t.bfloat16) -> None:
        super().__init__()
        pairs = head_dim // 2
        self.sections = [pairs - 2 * (pairs // 3), pairs // 3, pairs // 3]
        self.register_buffer("inv_freq", axis_frequencies(self.sections, base=100.0))
        self.query = nn.Parameter(0.02 * t.randn(width, dtype=dtype))
        self.blocks = nn.ModuleList(
            DecoderBlock(width, token_width, heads, kv_heads, head_dim, dtype)
            for _ in range(depth))
        self.norm_head = nn.Parameter(t.ones(width, dtype=dtype))
        self.head = nn.Linear(width, ATTRIBUTES)  # attributes are 32-bit
        nn.init.normal_(self.head.weight, std=0.02)
        nn.init.zeros_(self.head.bias)
        self._serve_eight_bits = False

    def serve_in_eight_bits(self, on: bool = True) -> None:
        """From here on, without gradients, the blocks' first network layer takes its input
        from ``rms_norm_residual_fp8`` and its weights in 8 bits with a scale per output; with
        ``on`` false, no longer.  The 8-bit weights are no part of the state: they follow the
        weights through further training, loading and moving.  Only a write through ``.data``
        without a forward with gradients before the next answer goes unseen: call this again."""
        self._serve_eight_bits = on
        for block in self.blocks:
            block.forget_eight_bit_weight()
            if on:
                block.eight_bit_weight()

    def forward(self, tokens: t.Tensor, token_pos: t.Tensor, query_pos: t.Tensor,
                key_lengths: t.Tensor | None = None,
                key_mask: t.Tensor | None = None) -> t.Tensor:
        """(B, L, 59) fp32 attributes.

        tokens (B, S, token_width), token_pos (S, 3) or (B, S, 3), query_pos (L, 3) or
        (B, L, 3): positions (view, row, column) in patches, integers or floats;
        key_lengths, key_mask as ``cross_attention`` takes them.
        """
        B, L = tokens.shape[0], query_pos.shape[-2]
        x = self.query.expand(B, L, -1).contiguous()
        residual = None
        eight = self._serve_eight_bits and not t.is_grad_enabled()
        for block in self.blocks:
            if t.is_grad_enabled():  # training may go on, by any means of writing the weights
                block.forget_eight_bit_weight()
            x, residual = block(x, residual, tokens, query_pos, token_pos, self.inv_freq,
                                self.sections, key_lengths, key_mask, eight)
        y, _ = rms_norm_residual(x, residual, self.norm_head)
        return self.head(y.float())


def to_gaussians(attributes: t.Tensor, query_pos: t.Tensor, view: dict, patch: int = 16,
                 depth: float = 3.0) -> gaussian:
    """The Gaussians of one view's queries: attributes (L, 59), query_pos (L, 3), whose rows and
    columns count patches.  Offsets, depths, scales and opacities are held within bounds (a
    patch to each side, ``depth`` e^+-1, e^+-2 of a quarter patch, logits +-4): a step of the
    optimizer moves all Gaussians at once and would otherwise drive them out of the image."""
    L = attributes.shape[0]
    a = attributes.split((2, 1, 4, 3, 1, 3, 45), dim=1)
    pixel = (query_pos[:, [2, 1]].float() + 0.5 + a[0].tanh()) * patch
    f = t.tensor([float(view["fx"]), float(view["fy"])], device=pixel.device)
    c = t.tensor([float(view["cx"]), float(view["cy"])], device=pixel.device)
    z = depth * a[1].tanh().exp()
    camera = t.cat(((pixel - c) / f * z, z), 1)
    g = gaussian(L)
    g.mu = ((camera - view["T"]) @ view["R"]).contiguous()  # R^T (x - t)
    g.q = a[2] + t.tensor([1.0, 0.0, 0.0, 0.0], device=pixel.device)
    g.s = 2.0 * a[3].tanh() + (0.25 * patch / float(view["fx"]) * z).log()
    g.alpha = 4.0 * a[4].tanh()
    g.A = a[5]
    g.k_j = a[6].reshape(L, 15, 3)
    return g
