"""Products added onto what is there (qmm_i8 with add=True), in every variant of the kernel: single blocks and pairs, columns shared by a cluster or
not, several tiles after one another.  Roundings: the product's three and the sum's, of half a step each, and for fp16 the last one."""
from __future__ import annotations

import numpy as np
import pytest

from tests import i8_formulas as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from vinf_3080ti_b200.runtime import Runtime

    r = Runtime()
    yield r
    r.synchronize()
    r.close()


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols,ntok", [(40000, 130, 20), (20001, 130, 77), (20000, 300, 300), (19997, 130, 1021), (3000, 512, 600), (513, 2050, 257), (5120, 17408, 8), (300, 9000, 4)])
def test_every_variant(rt, rows, cols, ntok, kind):
    rng = np.random.default_rng(rows + ntok)
    w, q = rng.integers(-128, 128, (rows, cols), dtype=np.int8), np.zeros((ntok, F.pitch(cols)), np.int8)
    q[:, :cols] = rng.integers(-128, 128, (ntok, cols), dtype=np.int8)
    ws, qs = rng.uniform(1e-6, 1e-4, rows).astype(np.float32), rng.uniform(1e-4, 1e-1, ntok).astype(np.float32)
    y0 = rng.standard_normal((ntok, rows)).astype(kind)
    rt.upload_i8("w", w, ws, cols, rows)
    for name, a in (("q", q), ("s", qs)):
        rt.alloc(name, a.size, a.dtype.itemsize)
        rt.write(name, a)
    rt.alloc("y", ntok * rows + 7, y0.dtype.itemsize)
    rt.write("y", np.concatenate([y0.ravel(), np.full(7, 3.0, kind)]))
    rt.qmm_i8("w", "q", "s", "y", ntok, add=True)
    y = rt.read_array("y")
    assert (y[ntok * rows:] == 3.0).all()
    # sums of at most 17408 * 2^14 < 2^53: exact in 64-bit floats
    v = (q[:, :cols].astype(np.float64) @ w.astype(np.float64).T) * qs.astype(np.float64)[:, None] * ws.astype(np.float64)
    want = y0.astype(np.float64) + v
    limit = 3 * 2.0**-24 * 1.01 * np.abs(v) + 2.0**-24 * 1.01 * np.abs(want) + (2.0**-11 * 1.01 * np.abs(want) + 2.0**-25 if kind is np.float16 else 0)
    off = np.abs(y[:ntok * rows].reshape(ntok, rows).astype(np.float64) - want) - limit
    assert (off <= 0).all(), np.argwhere(off > 0)[:5]
