"""The calls of several dependent launches (a mask's list, then attention and its join; delta and
zeros, the list, dk and dv, dq and their sums; the norm's backward and its weight's sum) on
another stream than the default, and captured in graphs: bit for bit the default stream's."""

from __future__ import annotations

import math

import pytest
import torch as t

pytestmark = pytest.mark.gpu

# few rows, rows and keys that are split into parts and joined, the widths of all kernels
SHAPES = [(2, 5, 900, 4, 2, 64), (2, 130, 1100, 8, 2, 64), (2, 130, 1100, 2, 1, 96),
          (1, 300, 2100, 2, 2, 128), (2, 3, 2100, 4, 1, 128)]


def _case(device, shape, name, seed):
    B, L, S, H, K, D = shape
    gen = t.Generator(device).manual_seed(seed)
    dtype = {"bf16": t.bfloat16, "fp16": t.float16}[name]
    randn = lambda *s: t.randn(*s, generator=gen, device=device).to(dtype)  # noqa: E731
    lengths = t.randint(S // 2, S + 1, (B,), generator=gen, device=device, dtype=t.int32)
    mask = t.rand(B, S, generator=gen, device=device) < (0.2 + 0.5 * (seed % 2))
    return [randn(B, L, H, D), randn(B, S, K, D), randn(B, S, K, D), randn(B, L, H, D), lengths, mask]


def _on_side_stream(call):
    """The call on another stream while the default one is busy, so that a launch sent there would
    be late."""
    busy = t.randn(2048, 2048, device="cuda")
    side = t.cuda.Stream()
    t.cuda.synchronize()
    for _ in range(20):
        busy = busy @ busy * 1e-3
    with t.cuda.stream(side):
        out = call()
        done = [x.clone() for x in out]
        side.synchronize()
    t.cuda.synchronize()
    return done


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_on_a_side_stream(device, shape, masked, name):
    from gaussian_splatting.decoder import cross_attention

    print(f"[gpu] side stream {shape} {masked} {name}", flush=True)
    q, k, v, do, lengths, mask = _case(device, shape, name, 1)

    def call():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        o = cross_attention(*leaves, key_lengths=lengths, key_mask=mask if masked else None)
        return [o.detach(), *t.autograd.grad(o, leaves, do)]

    want = [x.clone() for x in call()]
    for got in (_on_side_stream(call), _on_side_stream(call)):
        assert all(t.equal(a, b) for a, b in zip(got, want))


def _replays(held, cases, call):
    """Captures call() over `held`, whose contents then change from replay to replay, with eager
    work and synchronizations between."""
    want = []
    for case in cases:
        for x, y in zip(held, case):
            x.copy_(y)
        want.append([x.clone() for x in call()])
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        out = call()
    for turn in range(6):
        at = turn % len(cases)
        for x, y in zip(held, cases[at]):
            x.copy_(y)
        graph.replay()
        t.cuda.synchronize()
        assert all(t.equal(a, b) for a, b in zip(out, want[at])), turn
        eager = call()
        assert all(t.equal(a, b) for a, b in zip(eager, want[at])), turn


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_in_a_graph(device, crc, shape, masked, name):
    """Forward and backward in one graph, with other values, lengths and masks at each replay."""
    print(f"[gpu] graph {shape} {masked} {name}", flush=True)
    cases = [_case(device, shape, name, seed) for seed in (1, 2, 3)]
    held = [x.clone() for x in cases[0]]
    q, k, v, do, lengths, mask = held
    scale = 1 / math.sqrt(shape[5])

    def call():
        m = mask if masked else None
        o, lse, low = crc.cross_attention(q, k, v, lengths, m, scale, True)
        return [o, *crc.cross_attention_backward(do, q, k, v, o, lse, low, lengths, m, scale, True, True)]

    _replays(held, cases, call)


@pytest.mark.parametrize("rows,width", [(9, 100), (700, 1500), (3000, 5000)])
def test_norm_and_rotary_on_a_side_stream_and_in_a_graph(device, crc, rows, width):
    from gaussian_splatting.decoder import rms_norm_residual, rms_norm_residual_fp8

    print(f"[gpu] streams of the norm {rows} {width}", flush=True)

    def case(seed):
        gen = t.Generator(device).manual_seed(seed)
        randn = lambda *s: t.randn(*s, generator=gen, device=device).bfloat16()  # noqa: E731
        return [randn(rows, width), randn(rows, width), randn(width), randn(rows, width),
                randn(rows, width), randn(1, rows, 2, 16), t.rand(rows, 1, generator=gen, device=device)]

    held = [x.clone() for x in case(1)]
    x, r, w, dy, dh, z, pos = held
    inv = t.ones(8, device=device)

    def eager():
        leaves = [a.detach().requires_grad_(True) for a in (x, r, w)]
        y, h = rms_norm_residual(*leaves)
        with t.no_grad():
            y8, scale, _ = rms_norm_residual_fp8(x, r, w)
        return [y.detach(), h.detach(), *t.autograd.grad((y, h), leaves, (dy, dh)), y8.view(t.uint8),
                scale, crc.rotary_axes(z, pos, inv, [8], False, False)]

    want = [a.clone() for a in eager()]
    for got in (_on_side_stream(eager), _on_side_stream(eager)):
        assert all(t.equal(a, b) for a, b in zip(got, want))

    def raw():
        y, h, rstd = crc.rms_norm_residual(x, r, w, 1e-6, True)
        dx, dw = crc.rms_norm_residual_backward(h, rstd, w, dy, dh)
        y8, scale, _ = crc.rms_norm_residual_fp8(x, r, w, 1e-6)
        return [y, h, dx, dw, y8.view(t.uint8), scale, crc.rotary_axes(z, pos, inv, [8], False, True)]

    _replays(held, [case(1), case(2), case(3)], raw)
