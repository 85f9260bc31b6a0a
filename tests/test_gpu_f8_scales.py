"""Products whose scales' own product is at the ends of the range that the header gives for it, 2^-126 and 2^128, or 0.

Tolerances as in tests/test_gpu_f8.py.  Results may be subnormal: a block's part is added with a rounding of 2^-150 at most then, and there are as many as blocks of columns.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import f8_formulas as F
from tests.test_gpu_f8 import bound, put, put_rows, rt  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

# every variant of the kernel, with columns that are shared between blocks and without
SIZES = [(300, 700, 5), (1024, 5120, 4), (300, 700, 20), (1024, 5120, 20), (300, 700, 50), (1024, 5120, 50), (300, 700, 100), (1001, 4999, 177), (30000, 300, 130), (9000, 2000, 300),
         (1280, 10000, 600)]


def scales(rng, blocks, rows, row_blocks, low, high):
    """Of activations [blocks][rows] and weights [row_blocks][blocks], whose products' exponents lie between low and high + 1."""
    split = rng.integers(max(-140, low - 120), min(120, high + 140), blocks)  # of a block of columns: the activations' share
    each = rng.integers(0, (high - low) // 2 + 1, (blocks, rows))
    q = np.ldexp(rng.uniform(1, 1.4, (blocks, rows)), np.clip(split[:, None] + each, -149, 126))
    w = np.ldexp(rng.uniform(1, 1.4, (row_blocks, blocks)), np.clip(low - split[None] + rng.integers(0, (high - low) // 2 + 1, (row_blocks, blocks)), -149, 126))
    return q.astype(np.float32), w.astype(np.float32)


def product(rt, w, ws, q, qs):  # noqa: F811
    (rows, cols), ntok = w.shape, q.shape[0]
    rt.upload_f8("w8", w, ws, cols, rows)
    put_rows(rt, q, qs)
    put(rt, "y8", np.zeros(ntok * rows, np.float32))
    rt.qmm_f8("w8", "q8", "s8", "y8", ntok)
    rt.synchronize()
    return rt.read_array("y8").reshape(ntok, rows).astype(np.float64)


def check(rt, w, ws, q, qs):  # noqa: F811
    y = product(rt, w, ws, q, qs)
    want, most = F.qmm(w, ws, q, qs)
    assert np.abs(want).max() < 2.0**127
    off = np.abs(y - want) - bound(most, want, w.shape[1], np.float32) - F.blocks(w.shape[1]) * 2.0**-150
    assert (off <= 0).all(), (np.argwhere(~(off <= 0))[:5], y.flat[off.argmax()], want.flat[off.argmax()])
    return y


def values(rng, shape):
    b = rng.integers(0, 256, shape).astype(np.uint8)
    return np.where(b & 127 == 127, 0, b).astype(np.uint8)


@pytest.mark.parametrize("rows,cols,ntok", SIZES)
def test_products_of_scales_that_are_tiny(rt, rows, cols, ntok):  # noqa: F811
    rng = np.random.default_rng(rows + ntok)
    w, q = values(rng, (rows, cols)), values(rng, (ntok, cols))
    for low, high in ((-126, -110), (-124, -100), (-112, -90)):
        qs, ws = scales(rng, F.blocks(cols), ntok, F.blocks(rows), low, high)
        y = check(rt, w, ws, q, qs)
        assert (y != 0).any()


def few(rng, rows, cols, ntok):
    """Values of 2^-9, one for each activation row and block of columns."""
    q = np.zeros((ntok, F.blocks(cols) * F.BLOCK), np.uint8).reshape(ntok, -1, F.BLOCK)
    at = rng.integers(0, F.BLOCK, q.shape[:2] + (1,))
    np.put_along_axis(q, at, rng.choice([0, 1, 0x81], at.shape).astype(np.uint8), 2)
    return rng.choice([0, 0, 1, 0x81], (rows, cols)).astype(np.uint8), np.ascontiguousarray(q.reshape(ntok, -1)[:, :cols])


@pytest.mark.parametrize("rows,cols,ntok", SIZES)
def test_products_of_scales_that_are_huge(rt, rows, cols, ntok):  # noqa: F811
    """Sums of one product of 2^-18, or of none: zeros stay zeros."""
    rng = np.random.default_rng(rows + ntok)
    w, q = few(rng, rows, cols, ntok)
    for low, high in ((92, 106), (104, 124), (112, 126)):
        qs, ws = scales(rng, F.blocks(cols), ntok, F.blocks(rows), low, high)
        y = check(rt, w, ws, q, qs)
        assert (y != 0).any()


@pytest.mark.parametrize("rows,cols,ntok", SIZES)
def test_among_ordinary_ones(rt, rows, cols, ntok):  # noqa: F811
    """Some rows and some blocks of columns, zeros, one scale that is undefined, blocks of zeros whose scales are huge."""
    rng = np.random.default_rng(rows + ntok)
    blocks, row_blocks = F.blocks(cols), F.blocks(rows)
    w, q = values(rng, (rows, cols)), values(rng, (ntok, cols))
    qs = rng.uniform(0.01, 1, (blocks, ntok)).astype(np.float32)
    ws = rng.uniform(0.01, 1, (row_blocks, blocks)).astype(np.float32)
    some = rng.random((blocks, ntok))
    qs[some < 0.2] *= np.float32(2.0**-80)
    qs[some < 0.05] = 0
    ws[rng.random(ws.shape) < 0.2] *= np.float32(2.0**-30)
    last = blocks - 1
    q[:, last * F.BLOCK:] = 0
    qs[last], ws[:, last] = 2.0**100, 2.0**27
    check(rt, w, ws, q, qs)
    undefined = int(rng.integers(0, ntok))
    qs[0, undefined] = np.nan
    y = product(rt, w, ws, q, qs)
    assert np.isnan(y[undefined]).all()
    qs[0, undefined] = 0
    others = np.arange(ntok) != undefined
    want, most = F.qmm(w, ws, q, qs)
    assert (np.abs(y - want)[others] <= bound(most, want, cols, np.float32)[others]).all()
