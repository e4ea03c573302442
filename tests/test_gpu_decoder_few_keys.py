"""Scenes of few valid keys, alone or padded or masked to many: their results are off by their own
rounding and no more, since there are too few terms for the roundings of p and ds to average
out."""

from __future__ import annotations

import math

import pytest
import torch as t

import decoder_ref as ref

pytestmark = pytest.mark.gpu


def _case(shape, dtype, kind, few):
    B, L, S, H, K, D = shape
    gen = t.Generator().manual_seed(L + S + D)
    randn = lambda *s: t.randn(*s, generator=gen).to(dtype)  # noqa: E731
    q, k, v, do = randn(B, L, H, D), randn(B, S, K, D), randn(B, S, K, D), randn(B, L, H, D)
    lengths = mask = None
    if kind == "lengths":
        lengths = t.full((B,), S, dtype=t.int32)
        lengths[:len(few)] = t.tensor(few, dtype=t.int32)
    else:
        mask = t.ones(B, S, dtype=t.bool)
        for b, n in enumerate(few):
            mask[b] = False
            mask[b, t.randperm(S, generator=gen)[:n]] = True
    return q, k, v, do, lengths, mask


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["lengths", "keys"])
@pytest.mark.parametrize("shape", [(5, 130, 500, 4, 1, 64), (5, 200, 300, 2, 2, 96),
                                   (5, 90, 1100, 2, 1, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_few_valid_keys_among_many(device, shape, kind, name):
    """Batches of 2, 3, 64 and 0 valid keys beside a full one.  With up to 64 keys the errors of p
    and ds need not average out, so what their rounding leaves out is multiplied too: the bounds
    are the result's own rounding and the 32-bit terms, a quarter more of these for the u^2 of
    p, ds and o.  The full batch is held to the ordinary bounds."""
    print(f"[gpu] few valid keys {shape} {kind} {name}", flush=True)
    from gaussian_splatting.decoder import cross_attention

    dtype = ref.DTYPES[name]
    few = [2, 3, 64, 0]
    q, k, v, do, lengths, mask = _case(shape, dtype, kind, few)
    leaves = [x.to(device).requires_grad_(True) for x in (q, k, v)]
    on = lambda x: None if x is None else x.to(device)  # noqa: E731
    o = cross_attention(*leaves, key_lengths=on(lengths), key_mask=on(mask))
    got = dict(zip(("dq", "dk", "dv"), t.autograd.grad(o, leaves, do.to(device))), o=o)
    want, wide = ref.attention(q, k, v, do, lengths, mask)
    _, tight = ref.attention(q, k, v, do, lengths, mask, dtype=t.float32)
    n = len(few)
    for what, x in got.items():
        ref.assert_within(x[n:], want[what][n:], wide[what][n:], what)
        bound = ref.U[dtype] * want[what].abs() + ref.TINY[dtype] + 1.25 * tight[what]
        ref.assert_within(x[:n], want[what][:n], bound[:n], what)


@pytest.mark.parametrize("kind", ["lengths", "keys"])
def test_a_padded_scene_answers_as_it_does_alone(device, kind):
    """Two keys alone and the same two among 700: the errors against 64 bits are of one size (the
    sums' orders differ, so not bit for bit), a fifth at most apart."""
    from gaussian_splatting.decoder import cross_attention

    shape = (1, 300, 700, 2, 2, 64)
    q, k, v, do, lengths, mask = _case(shape, t.bfloat16, kind, [2])
    at = ref.valid_of(1, 700, lengths, mask)[0].nonzero()[:, 0]
    want, _ = ref.attention(q, k, v, do, lengths, mask)

    def errors(k, v, at, **kw):
        leaves = [x.to(device).requires_grad_(True) for x in (q, k, v)]
        o = cross_attention(*leaves, **kw)
        dq, dk, dv = t.autograd.grad(o, leaves, do.to(device))
        pairs = ((o, want["o"]), (dq, want["dq"]), (dk[:, at], want["dk"][:, valid]),
                 (dv[:, at], want["dv"][:, valid]))
        return [float((ref.f64(a) - b).norm()) for a, b in pairs]

    valid = at
    alone = errors(k[:, at], v[:, at], slice(None))
    among = errors(k, v, at.to(device), key_lengths=None if lengths is None else lengths.to(device),
                   key_mask=None if mask is None else mask.to(device))
    for a, b in zip(alone, among):
        assert b <= 1.2 * a + 1e-12, (alone, among)
    assert math.isfinite(sum(among))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_gradients_of_one_row_against_few_keys(device, dim, name):
    """Only the first of 500 rows has a gradient, so dk_j = ds_j q: every value is off by its own
    rounding, U at most, and so is their factor on q.  A tenth more for 32-bit terms.  delta is
    formed from an o whose p are not rounded, so that small ds do not carry that."""
    from gaussian_splatting.decoder import cross_attention

    print(f"[gpu] one row's gradients, few keys {dim} {name}", flush=True)
    gen = t.Generator(device).manual_seed(7)
    randn = lambda *s: t.randn(*s, generator=gen, device=device)  # noqa: E731
    q, k, v = (randn(2, n, 2, dim).to(ref.DTYPES[name]) for n in (500, 60, 60))
    do = t.zeros_like(q)
    do[:, 0] = (256 * randn(2, 2, dim)).to(q.dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    _, dk, _ = t.autograd.grad(cross_attention(*leaves), leaves, do)
    for b in range(2):
        for h in range(2):
            qq, kk, vv, g = (x.detach().double() for x in (q[b, 0, h], k[b, :, h], v[b, :, h], do[b, 0, h]))
            p = (kk @ qq / math.sqrt(dim)).softmax(0)
            dp = vv @ g
            ds = p * (dp - p @ dp) / math.sqrt(dim)
            have = dk[b, :, h].double() @ qq / (qq @ qq)
            large = ds.abs() >= ds.abs().median()
            off = ((have - ds).abs() / ds.abs() / ref.U[q.dtype])[large]
            assert float(off.max()) <= 1.1, (b, h, float(off.max()))


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("queries", [1, 16, 400])
@pytest.mark.parametrize("keys", [2, 33, 64])
def test_o_of_few_keys_is_rounded_once(device, keys, queries, name):
    """The output's own rounding and the 32-bit terms, a quarter more of these for the u^2 of p."""
    print(f"[gpu] o of few keys {keys} {queries} {name}", flush=True)
    from gaussian_splatting.decoder import cross_attention

    dtype = ref.DTYPES[name]
    for dim in (40, 96, 128):
        q, k, v, _, _, _ = _case((3, queries, keys, 4, 2, dim), dtype, "lengths", [])
        o = cross_attention(q.to(device), k.to(device), v.to(device))
        want, tight = ref.attention(q, k, v, dtype=t.float32)
        bound = ref.U[dtype] * want["o"].abs() + ref.TINY[dtype] + 1.25 * tight["o"]
        ref.assert_within(o, want["o"], bound, f"o {dim}")
