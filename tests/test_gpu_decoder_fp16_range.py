"""Gradients of cross attention in fp16 over the type's range: values of any size, rows whose
gradients differ by orders, and heads near the largest value."""

from __future__ import annotations

import math

import pytest
import torch as t

pytestmark = pytest.mark.gpu

U = 2.0 ** -11  # fp16's rounding, relative; 2^-25 below its normal range


def _exact(q, k, v, do, valid=None):
    """dq, dk, dv from the definition in 64 bits on the device."""
    (B, L, H, D), (S, K) = q.shape, k.shape[1:3]
    q, k, v, do = (x.detach().double() for x in (q, k, v, do))
    dq, dk, dv = (t.zeros_like(x) for x in (q, k, v))
    for b in range(B):
        at = (t.ones(S, dtype=t.bool, device=q.device) if valid is None else valid[b]).nonzero()[:, 0]
        for h in range(H):
            j = h // (H // K)
            kk, vv = k[b, at, j], v[b, at, j]
            p = (q[b, :, h] @ kk.T / math.sqrt(D)).softmax(-1)
            g = do[b, :, h]
            ds = p * (g @ vv.T - (g * (p @ vv)).sum(-1, keepdim=True)) / math.sqrt(D)
            dq[b, :, h] = ds @ kk
            dk[b, at, j] += ds.T @ q[b, :, h]
            dv[b, at, j] += p.T @ g
    return dq, dk, dv


def _gradients(q, k, v, do, **kw):
    from gaussian_splatting.decoder import cross_attention

    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    return t.autograd.grad(cross_attention(*leaves, **kw), leaves, do)


def _assert_rows(got, want, factor, what, names=("dq", "dk", "dv")):
    """The error of every row of `dim` values, as a norm, within factor times what rounding
    moves at most: U of the row, and 2^-25 of each value below the type's normal range."""
    for g, w, n in zip(got, want, ("dq", "dk", "dv")):
        if n not in names:
            continue
        assert g.isfinite().all(), (what, n)
        error = (g.double() - w).norm(dim=-1)
        bound = factor * U * w.norm(dim=-1) + 2.0 ** -25 * math.sqrt(w.shape[-1])
        worst = float((error / bound).max())
        assert worst <= 1.0, f"{what} {n}: {worst:.2f} times the bound"


def _randn(device, seed):
    gen = t.Generator(device).manual_seed(seed)
    return lambda *s: t.randn(*s, generator=gen, device=device)


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("value", [1100.0, 30000.0])
def test_values_near_the_largest_do_not_overflow(device, value, dim):
    """Two keys of equal score and opposite values: ds is half of do.v, which the type holds
    only scaled down.  Each gradient is a sum of two terms, ds k with ds rounded to the type and
    then to itself: |k1| + |k2| is up to about twice |k1 - k2|, so three roundings."""
    print(f"[gpu] fp16 range, values {value} dim {dim}", flush=True)
    randn = _randn(device, dim)
    q = t.zeros(1, 3, 1, dim, device=device).half()
    k = randn(1, 2, 1, dim).half()
    v = t.tensor([1.0, -1.0], device=device)[None, :, None, None].mul(value).half().expand(1, 2, 1, dim)
    q[0, 1:] = 1e-3
    k[0, 1] = -k[0, 0]
    # the scores are equal: q is constant and k's halves cancel
    k[..., dim // 2:] = -k[..., :dim // 2]
    do = t.full_like(q, 1e-3)
    _assert_rows(_gradients(q, k, v, do), _exact(q, k, v, do), 3.0, (value, dim))


@pytest.mark.parametrize("L,S,H,K,D", [(40, 8160, 2, 1, 64), (100, 8160, 2, 1, 64),
                                       (80, 32400, 1, 1, 128), (70, 4100, 3, 1, 96)])
@pytest.mark.parametrize("size", [0.01, 0.02, 1.0, 4000.0])
def test_values_of_any_size_keep_the_gradients_digits(device, size, L, S, H, K, D):
    """Thousands of keys, each p about 1 / S, and values of size `size`.  A row's rounding and
    that of its terms are each 0.42 U in the mean (uniform over a binade) and independent: 0.6 U
    together, for which 1.5 leaves room (a norm over 64 values varies by a tenth).  dv has no
    rounded factor but p, with the same count."""
    print(f"[gpu] fp16 range {size} {(L, S, H, K, D)}", flush=True)
    randn = _randn(device, S + D)
    q, k, do = randn(1, L, H, D).half(), randn(1, S, K, D).half(), randn(1, L, H, D).half()
    v = (size * randn(1, S, K, D)).half()
    # dk is a sum over L H / K rows alone, of one key's p: its terms average out all the same
    _assert_rows(_gradients(q, k, v, do), _exact(q, k, v, do), 1.5, (size, L, S, H, K, D))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("L,S,H,K,D", [(24, 8160, 2, 2, 64), (100, 4100, 4, 2, 128)])
def test_rows_of_unequal_gradients_keep_their_digits(device, L, S, H, K, D, masked):
    """Row i's do is 2^-(i mod 13) of the largest, as for Gaussians seen and nearly hidden: every
    row's dq is as near as the largest's.  Masked keys hold values that would set any scale."""
    print(f"[gpu] fp16 range, unequal rows {(L, S, H, K, D)} {masked}", flush=True)
    randn = _randn(device, L)
    q, k, v = randn(2, L, H, D).half(), randn(2, S, K, D).half(), randn(2, S, K, D).half()
    do = (randn(2, L, H, D) * 2.0 ** -(t.arange(L, device=device) % 13).float()[:, None, None]).half()
    mask = None
    if masked:
        mask = t.rand(2, S, generator=t.Generator(device).manual_seed(2), device=device) < 0.7
        v = v.masked_fill(~mask[:, :, None, None], 65504.0)
    got = _gradients(q, k, v, do, key_mask=mask)
    _assert_rows(got, _exact(q, k, v, do, mask), 1.5, (L, S, masked))


@pytest.mark.parametrize("D", [64, 128])
def test_keys_that_only_rows_of_small_gradients_read(device, D):
    """Row r reads keys 2r and 2r + 1 alone (the others' scores lie 20 or more below), and its do is
    2^-(r mod 17) of the largest: dk and dv of those keys keep their digits too.  dk is one term, ds
    q: a rounding of its own and one of ds; delta carries what p's rounding in the forward moved o
    by, half of one where the two values are opposite; 32-bit scores of 2^7 (in powers of two) are
    off by 2^-16.  Three in all; dq, the difference of two like keys, is not compared."""
    print(f"[gpu] fp16 range, keys of small rows {D}", flush=True)
    R = 100
    randn = _randn(device, D)
    unit = randn(R, D)
    unit = unit / unit.norm(dim=-1, keepdim=True)
    # q_r.k_2r / sqrt(D) = 60 for its own, at most 0.6 of that for other rows' keys
    q = (unit * math.sqrt(60 * math.sqrt(D)))[None, :, None].half()
    k = q.repeat_interleave(2, 1).contiguous()
    k[:, 1::2] += (0.05 * randn(1, R, 1, D)).half()
    v = randn(1, 2 * R, 1, D).half()
    v[:, 1::2] = -v[:, ::2]
    small = 2.0 ** -(t.arange(R, device=device) % 17).float()[:, None, None]
    do = (16 * randn(1, R, 1, D) * small).half()
    _assert_rows(_gradients(q, k, v, do), _exact(q, k, v, do), 3.0, D, names=("dk", "dv"))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_row_whose_gradient_is_not_finite_leaves_the_others_dq(device, bad, name):
    """Bit for bit: the scale that ds is rounded at is each row's own."""
    dtype = {"bf16": t.bfloat16, "fp16": t.float16}[name]
    for L, D in ((20, 64), (150, 128)):
        randn = _randn(device, L)
        q, k, v, do = (randn(1, n, 2, D).to(dtype) for n in (L, 300, 300, L))
        clean = _gradients(q, k, v, do)[0]
        broken = do.clone()
        broken[0, 7, 1, 3] = bad
        got = _gradients(q, k, v, broken)[0]
        rest = t.ones(1, L, 2, dtype=t.bool, device=device)
        rest[0, 7, 1] = False
        assert got[~rest].isnan().all()
        assert t.equal(got[rest], clean[rest])


@pytest.mark.parametrize("size", [1e-6, 2.0 ** 12])
@pytest.mark.parametrize("L,S,D", [(100, 300, 64), (40, 1200, 128)])
def test_gradients_of_a_mean_and_of_a_scaled_loss(device, size, L, S, D):
    """do of 1e-6, itself below the type's normal range, and of 2^12."""
    print(f"[gpu] fp16 range, do of {size} {(L, S, D)}", flush=True)
    randn = _randn(device, L)
    q, k, v = randn(1, L, 2, D).half(), randn(1, S, 2, D).half(), randn(1, S, 2, D).half()
    do = (size * randn(1, L, 2, D)).half()
    _assert_rows(_gradients(q, k, v, do), _exact(q, k, v, do), 1.5, (size, L, S, D))
