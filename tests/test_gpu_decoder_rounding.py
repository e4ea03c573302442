"""What the rounding of a 32-bit value to the type leaves out, where the attention kernels keep
it: the two parts add up to the value, at every value."""

from __future__ import annotations

import math

import pytest
import torch as t

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
DTYPES = {"bf16": t.bfloat16, "fp16": t.float16}


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("queries", [1, 40, 300])
@pytest.mark.parametrize("keys", [3, 700])
def test_o_and_its_low_part_add_up(device, queries, keys, name):
    """Three valid keys of equal score: p is exact in the products, so o is the mean of three
    values in 32 bits.  o + o_low holds 2^-20 of it (two significands of 8 bits hold 2^-16), and
    2^-24 below fp16's normal range."""
    import custom_rasterizer_cuda as crc

    print(f"[gpu] low part of o {queries} {keys} {name}", flush=True)
    gen = t.Generator(device).manual_seed(queries + keys)
    B, K, D = 2, 64, 128
    q = t.zeros(B, queries, K, D, device=device, dtype=DTYPES[name])
    k = t.randn(B, keys, K, D, generator=gen, device=device).to(q.dtype)
    v = t.randn(B, keys, K, D, generator=gen, device=device).to(q.dtype)
    lengths = t.full((B,), 3, dtype=t.int32, device=device)
    o, _, low = crc.cross_attention(q, k, v, lengths, None, 0.1, True)
    want = v[:, :3].double().mean(1, keepdim=True).expand_as(o)
    bound = want.abs() * (2.0 ** -20 if name == "fp16" else 2.0 ** -15) + 2.0 ** -24
    # 32-bit sums of three terms whose sizes may cancel
    bound = bound + 2.0 ** -22 * v[:, :3].double().abs().mean(1, keepdim=True)
    error = (o.double() + low.double() - want).abs()
    assert bool((error <= bound).all()), float((error / bound).max())


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("queries,keys", [(1, 8160), (24, 8160)])
def test_gradients_of_one_row_are_rounded_once(device, queries, keys, dim, name):
    """Only the first row of each head has a gradient, so dk_j = ds_j q: with what ds's rounding
    leaves out multiplied too, every value of dk is off by its own rounding, U at most, and so
    is their factor on q.  A tenth more for delta, whose o carries p's rounding in the forward
    (0.3 U p each, independent: 1e-2 of U for keys whose ds is not among the smaller half), and
    for 32-bit terms.  dv_j = p_j do likewise; dq with do = 0 elsewhere is 0 there."""
    from gaussian_splatting.decoder import cross_attention

    print(f"[gpu] one row's gradients {queries} {keys} {dim} {name}", flush=True)
    gen = t.Generator(device).manual_seed(7)
    randn = lambda *s: t.randn(*s, generator=gen, device=device)  # noqa: E731
    B, K = 2, 2
    q, k, v = (randn(B, n, K, dim).to(DTYPES[name]) for n in (queries, keys, keys))
    do = t.zeros_like(q)
    do[:, 0] = (256 * randn(B, K, dim)).to(q.dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    dq, dk, dv = t.autograd.grad(cross_attention(*leaves), leaves, do)
    assert (dq[:, 1:] == 0).all()
    for b in range(B):
        for h in range(K):
            qq, kk, vv, g = (x.detach().double() for x in (q[b, 0, h], k[b, :, h], v[b, :, h], do[b, 0, h]))
            p = (kk @ qq / math.sqrt(dim)).softmax(0)
            dp = vv @ g
            ds = p * (dp - p @ dp) / math.sqrt(dim)
            for got, factor, row, what in ((dk, ds, qq, "dk"), (dv, p, g, "dv")):
                # the factor that the gradient's rows hold, against the exact one
                have = got[b, :, h].double() @ row / (row @ row)
                # values of the type's normal range: the row's root mean square well inside it
                size = factor.abs()
                large = (size >= size.median()) & (size * row.norm() / math.sqrt(dim) > 2.0 ** -11)
                assert int(large.sum()) >= keys // 4
                off = ((have - factor).abs() / size / U[name])[large]
                assert float(off.max()) <= 1.1, (what, b, h, float(off.max()))
