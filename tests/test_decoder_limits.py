"""Calls whose launches would hold 2^32 work-items are refused by the host, with a message, before
any HIP call (here, without a device, a launch would be HIP's error)."""

from __future__ import annotations

import ctypes as c
from pathlib import Path

import pytest

import decoder_abi as abi

LIB = Path(__file__).resolve().parents[1] / "custom-3dgs-cuda_amd" / "libgsrdecoder.so"
P = abi.P


@pytest.fixture(scope="module")
def lib():
    assert LIB.exists(), "libgsrdecoder.so is not built (python custom-3dgs-cuda_amd/build.py)"
    return abi.load(LIB)


def _refused(lib, rc, word):
    assert rc == abi.INVALID and word in lib.gsd_last_error(), (rc, lib.gsd_last_error())


def test_forward(lib):
    # a work-group of 256 for each batch and key head, or each 128 rows of one
    for kw in (dict(batch=2 ** 24, heads=1, kv_heads=1, queries=1, keys=1),
               dict(batch=2 ** 21, heads=8, kv_heads=8, queries=3, keys=5),
               dict(batch=2 ** 12, heads=1, kv_heads=1, queries=2 ** 19, keys=5)):
        a = abi.attention(dim=8, **kw)
        _refused(lib, lib.gsd_cross_attention(c.byref(a), P, 2 ** 62, None), b"rows")


def test_backward(lib):
    grad = abi.AttentionGrad(d_o=P, do_stride_l=256, do_stride_h=64, dq=P, dk=P, dv=P)
    for dtype in (abi.BF16, abi.F16):
        # rows, keys, and the zeros of keys that take no part (2048 values of dk and dv each)
        for kw in (dict(batch=2 ** 24, heads=1, kv_heads=1, queries=1, keys=1, dim=8),
                   dict(batch=2 ** 14, heads=1, kv_heads=1, queries=1, keys=2 ** 17, dim=8),
                   dict(batch=2 ** 11, heads=1, kv_heads=1, queries=1, keys=2 ** 17, dim=128)):
            a = abi.attention(dtype=dtype, **kw)
            _refused(lib, lib.gsd_cross_attention_backward(c.byref(a), c.byref(grad), P, 2 ** 62, None),
                     b"too many")


def test_masks(lib):
    a = abi.attention(batch=2 ** 22, heads=1, kv_heads=1, queries=1, keys=1, dim=8, key_mask=P)
    _refused(lib, lib.gsd_cross_attention(c.byref(a), P, 2 ** 62, None), b"batch")


def test_rotary(lib):
    a = abi.rotary(batch=2 ** 15, length=2 ** 15, heads=1, dim=8, sections=(2, 2))
    _refused(lib, lib.gsd_rotary_axes(c.byref(a), None), b"large")
