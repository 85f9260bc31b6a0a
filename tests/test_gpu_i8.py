"""Passes in 8-bit integers on the GPU against their formulas in 64 bits (tests/i8_formulas.py).

Tolerances.  Integers and the choice of an integer are exact.  A product is float(sum) * scale * scale: three roundings of at most half a step
each, 3 * 2^-24 relative, an fp16 output one more of 2^-11 (2^-25 absolute among its subnormals); the second-order terms are within 1 %.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import i8_formulas as F
from vinf_3080ti_b200.gguf_types import GGUFTensorType as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt(codebooks):
    from vinf_3080ti_b200.runtime import Runtime

    r = Runtime(codebooks["iq3s_grid"], codebooks)
    yield r
    r.synchronize()
    r.close()


def put(rt, name, a):
    a = np.ascontiguousarray(a)
    rt.alloc(name, a.size, a.dtype.itemsize)
    rt.write(name, a)


def run_rows(rt, x, *, x2=None, residual=None, norm=None, eps=1e-6, total=None):
    ntok, cols = x.shape
    put(rt, "x", x)
    rt.alloc("q", ntok * F.pitch(cols) + 16, 1)
    rt.write("q", np.full(ntok * F.pitch(cols) + 16, 99, np.int8))
    put(rt, "s", np.full(ntok + 1, 7.0, np.float32))
    if x2 is not None:
        put(rt, "x2", x2)
    if residual is not None:
        put(rt, "r", residual)
        if total == "t":
            put(rt, "t", np.zeros_like(x))
    if norm is not None:
        put(rt, "g", norm)
    rt.rows_i8("x", "q", "s", cols, ntok, residual=None if residual is None else "r", total=total, norm=None if norm is None else "g", eps=eps,
               silu_mul=None if x2 is None else "x2")
    rt.synchronize()
    q = rt.read_array("q")
    assert (q[ntok * F.pitch(cols):] == 99).all()  # nothing behind the last row
    q = q[:ntok * F.pitch(cols)].reshape(ntok, F.pitch(cols))
    assert (q[:, cols:] == 0).all()
    s = rt.read_array("s")
    assert s[ntok] == 7.0
    got_total = None if residual is None else rt.read_array(total or "r").reshape(ntok, cols)
    return q[:, :cols], s[:ntok], got_total


def check_rows(rt, x, **kw):
    total = kw.pop("total", None)
    q, s, t = run_rows(rt, x, total=total, **kw)
    want_q, want_s, want_t = F.rows_i8(x, **kw)
    assert np.array_equal(s, want_s, equal_nan=True)
    assert np.array_equal(q, want_q), np.argwhere(q != want_q)[:5]
    if want_t is not None:
        assert np.array_equal(t, want_t, equal_nan=True)


COLS = [1, 2, 3, 15, 16, 17, 64, 127, 255, 1000, 2047, 2048, 4099, 5120, 8200, 17408]


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("cols", COLS)
def test_rows_of_every_length(rt, cols, kind):
    rng = np.random.default_rng(cols)
    for ntok in (1, 3, 5):
        x = (rng.standard_normal((ntok, cols)) * 2).astype(kind)
        x[:, 0] *= 20
        res = (rng.standard_normal((ntok, cols)) * 3).astype(kind)
        x2 = rng.standard_normal((ntok, cols)).astype(kind)
        g = rng.uniform(0.5, 1.5, cols).astype(np.float32)
        check_rows(rt, x)
        check_rows(rt, x, norm=g, eps=1e-5)
        check_rows(rt, x, residual=res, norm=g)
        check_rows(rt, x, residual=res, norm=g, total="t")
        check_rows(rt, x, residual=res, total="x")
        check_rows(rt, x, x2=x2)
        check_rows(rt, x, x2=x2, norm=g, eps=0.0)


@pytest.mark.parametrize("cols", [32768, 40001, 131071])
def test_long_rows(rt, cols):
    rng = np.random.default_rng(cols)
    x, res = rng.standard_normal((2, 2, cols)).astype(np.float32)
    g = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    check_rows(rt, x, residual=res, norm=g)
    check_rows(rt, x, x2=res)


@pytest.mark.parametrize("ntok,cols", [(700, 520), (3000, 64), (149, 5120)])
def test_many_rows(rt, ntok, cols):
    rng = np.random.default_rng(ntok)
    x, res = rng.standard_normal((2, ntok, cols)).astype(np.float32)
    check_rows(rt, x, residual=res, norm=rng.uniform(0.5, 1.5, cols).astype(np.float32), total="t")


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("cols", [1, 5, 33, 997, 1023, 1025, 2047, 4095, 4097, 5121, 6138, 6139, 6142, 8191])
def test_many_rows_of_any_length(rt, cols, kind):
    """More rows than SMs; rows that begin anywhere on a line."""
    rng = np.random.default_rng(cols)
    ntok = 203
    x, res = (rng.standard_normal((2, ntok, cols)) * 2).astype(kind)
    g = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    check_rows(rt, x, residual=res, norm=g)
    check_rows(rt, x, residual=res, norm=g, total="t")
    check_rows(rt, x)
    check_rows(rt, x, x2=res)
    check_rows(rt, x, x2=res, norm=g)


@pytest.mark.parametrize("cols,ntok", [(12282, 170), (12283, 170), (12288, 1), (20464, 2), (20481, 2), (20496, 160), (24560, 3), (24564, 3), (24565, 3), (24568, 150)])
def test_lengths_at_which_another_kernel_takes_over(rt, cols, ntok):
    rng = np.random.default_rng(cols)
    x, res = rng.standard_normal((2, ntok, cols)).astype(np.float32)
    g = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    check_rows(rt, x, residual=res, norm=g)
    check_rows(rt, x[:5], x2=res[:5])
    check_rows(rt, x[:5], x2=res[:5], norm=g)


def test_equal_largest_values_and_equal_rows(rt):
    """The largest product more than once: in one thread's vectors, in several; products that round to the same 32 bits."""
    rng = np.random.default_rng(12)
    for cols in (64, 5120, 5121, 20000):
        x = np.full((3, cols), 0.7, np.float32)
        x[1] = rng.choice(np.float32([0.1, -0.3, 0.3]), cols)
        g = np.full(cols, 1.3, np.float32)
        g[cols // 2:] = np.nextafter(np.float32(1.3), np.float32(2))
        x[2] = np.where(np.arange(cols) < cols // 2, np.float32(0.9), np.nextafter(np.float32(0.9), np.float32(0)))
        check_rows(rt, x, norm=g, eps=1e-3)
        check_rows(rt, x, x2=np.ascontiguousarray(x[:, ::-1]))
        check_rows(rt, x)


def test_gated_values_far_from_zero(rt):
    """Large negative x, whose silu is all but nothing, beside ordinary ones and beside large x2."""
    rng = np.random.default_rng(13)
    x = np.concatenate([np.linspace(-120, 120, 601), [-88.5, -87.0, -103.0, -200.0, 1e4, -1e4]]).astype(np.float32)
    x = np.tile(x, (6, 1))
    x2 = rng.standard_normal(x.shape).astype(np.float32)
    x[1] = np.minimum(x[1], -79)
    x[2] = np.minimum(x[2], -95)
    x2[3, ::7] = 1e20
    x2[4] *= np.float32(1e-25)
    x[5, x[5] > -60] = 0
    x2[5, ::5] = 1e30
    check_rows(rt, x, x2=x2)
    check_rows(rt, x, x2=x2, norm=np.ones(x.shape[1], np.float32))
    check_rows(rt, np.tile(x, (40, 1)), x2=np.tile(x2, (40, 1)))


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_halves_go_to_even(rt, kind):
    x = np.zeros((2, 260), kind)
    x[0, :127], x[0, 127] = np.arange(127) + 0.5, 127  # scale 1
    x[0, 128:255] = -(np.arange(127) + 0.5)
    x[1, :127], x[1, 127] = (np.arange(127) + 0.5) / 8, 127 / 8
    q, s, _ = run_rows(rt, x)
    assert s.tolist() == [1.0, 0.125]
    want = np.rint(np.arange(127) + 0.5)
    assert np.array_equal(q[0, :127], want) and np.array_equal(q[0, 128:255], -want) and np.array_equal(q[1, :127], want)
    check_rows(rt, x)


def test_values_next_to_a_half_are_decided_exactly(rt):
    """Scale 1, values one fp32 step to either side of k + 1/2."""
    k = np.arange(126, dtype=np.float32) + np.float32(0.5)
    x = np.concatenate([k, np.nextafter(k, np.float32(1e9)), np.nextafter(k, np.float32(-1e9)), [127.0]]).astype(np.float32)[None]
    check_rows(rt, x)
    # and after a norm whose factor is not a power of two: many rows, so that some values come close
    rng = np.random.default_rng(3)
    check_rows(rt, rng.standard_normal((400, 1024)).astype(np.float32), norm=np.full(1024, 1.1, np.float32), eps=0.1)


def test_zero_tiny_and_huge_rows(rt):
    x = np.zeros((8, 96), np.float32)
    x[1, 5] = 1e-44       # scale rounds to a subnormal or to zero
    x[2] = 1e-38
    x[3, ::2] = 3e38      # squares beyond fp32
    x[4, 1] = -3.4e38
    x[5] = np.float32(1e-30)
    x[6, 0], x[6, 1] = 1.0, 1e-30
    x[7] = -5.0
    check_rows(rt, x)
    check_rows(rt, x, norm=np.ones(96, np.float32), eps=1e-6)
    check_rows(rt, x, x2=np.ones((8, 96), np.float32))


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("ntok", [3, 150])
@pytest.mark.parametrize("cols", [1018, 1019, 1024, 1028, 4090, 4091, 4096, 4100, 5120, 5121, 6138, 6140, 10232, 10234, 10236, 12281, 12284, 16384, 17406, 18432, 18435, 20474, 20480, 24563])
def test_lengths_and_numbers_of_rows_at_which_blocks_change(rt, cols, ntok, kind):
    rng = np.random.default_rng(cols + ntok)
    x, y = (rng.standard_normal((ntok, cols)).astype(kind) for _ in range(2))
    check_rows(rt, x, residual=y, norm=rng.uniform(0.5, 1.5, cols).astype(np.float32), total="t")
    check_rows(rt, x, x2=y)


def test_gates_that_are_subnormal_or_far_below_zero(rt):
    """Their sigmoid or their product with it has few digits left, their values count all the same."""
    rng = np.random.default_rng(8)
    for low, high, size in ((1e-42, 1e-39, 1e30), (1e-38, 1e-37, 1e28), (-79.9, -60.0, 1e32), (-80.0, -1.0, 1.0), (-120.0, -70.0, 1e3), (-85.0, -79.0, 2e3)):
        x = rng.uniform(low, high, (30, 999)).astype(np.float32)
        check_rows(rt, x, x2=(rng.standard_normal((30, 999)) * size).astype(np.float32))


@pytest.mark.parametrize("cols", [64, 67, 1536])
def test_norms_of_values_at_the_ends_of_fp32(rt, cols):
    """Root mean squares whose reciprocal fp32 does not hold, and weights that bring the products back."""
    rng = np.random.default_rng(cols)
    g = rng.uniform(0.5, 1.5, cols)
    x = rng.standard_normal((40, cols))
    for size, weight in ((1e-40, 1e20), (1e-38, 1e18), (1e-42, 1e30), (8e37, 1e-20), (8e37, 1e-8), (3e37, 1.0)):
        check_rows(rt, (x.clip(-4, 4) * size).astype(np.float32), norm=(g * weight).astype(np.float32), eps=0.0)


def test_undefined_rows_have_an_undefined_scale_and_leave_the_others_alone(rt):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 333)).astype(np.float32)
    x[1, 7], x[2, 332], x[4, 0] = np.nan, np.inf, -np.inf
    g = np.ones(333, np.float32)
    for kw in ({}, {"norm": g}, {"residual": np.ones_like(x)}, {"residual": np.ones_like(x), "norm": g}):
        check_rows(rt, x, **kw)
        assert np.isnan(rt.read_array("s")[:6]).tolist() == [False, True, True, False, True, False]
    check_rows(rt, x, norm=np.full(333, np.inf, np.float32))
    # a scale beyond fp32
    big = np.full((2, 48), 3e38, np.float32)
    check_rows(rt, big, x2=np.full((2, 48), 1e30, np.float32))
    # silu of large negative values is zero, of -inf undefined
    low = np.full((2, 48), -1e4, np.float32)
    low[1, 3] = -np.inf
    check_rows(rt, low, x2=np.ones((2, 48), np.float32))
    # fp16 sums beyond 65504 are infinite
    half = np.full((1, 40), 60000, np.float16)
    check_rows(rt, half, residual=half)


def test_norm_weights_may_be_a_tensor(rt):
    rng = np.random.default_rng(8)
    g = rng.uniform(0.5, 1.5, 128).astype(np.float32)
    x = rng.standard_normal((3, 128)).astype(np.float32)
    rt.upload("gain", g, int(T.F32), 128, 1)
    put(rt, "x", x)
    rt.alloc("q", 3 * 128, 1)
    rt.alloc("s", 3)
    rt.rows_i8("x", "q", "s", 128, 3, norm="gain")
    want_q, want_s, _ = F.rows_i8(x, norm=g)
    assert np.array_equal(rt.read_array("q").reshape(3, 128), want_q) and np.array_equal(rt.read_array("s"), want_s)


# ---- the product ------------------------------------------------------------------------------------------------------


def make(rng, rows, cols, ntok, extreme=False):
    w = np.full((rows, cols), -128, np.int8) if extreme else rng.integers(-128, 128, (rows, cols), dtype=np.int8)
    q = np.full((ntok, cols), -128, np.int8) if extreme else rng.integers(-128, 128, (ntok, cols), dtype=np.int8)
    return w, rng.uniform(1e-4, 1e-2, rows).astype(np.float32), q, rng.uniform(1e-4, 1e-1, ntok).astype(np.float32)


def put_q(rt, name, q, junk=77):
    """Rows at their pitch; what lies behind a row's columns is not zero."""
    full = np.full((q.shape[0], F.pitch(q.shape[1])), junk, np.int8)
    full[:, :q.shape[1]] = q
    put(rt, name, full)


def bound(want, kind, extra=0.0):
    b = (3 * 2.0**-24 * 1.01 + extra) * np.abs(want)
    return b + 2.0**-11 * 1.01 * np.abs(want) + 2.0**-25 if kind is np.float16 else b + 2.0**-149


def check_product(rt, w, ws, q, qs, kind=np.float32, bind=None):
    (rows, cols), ntok = w.shape, q.shape[0]
    if bind is None:
        rt.upload_i8("w8", w, ws, cols, rows)
    put_q(rt, "q8", q)
    put(rt, "s8", qs)
    fill = np.full(ntok * rows + 5, 3.0, kind)
    put(rt, "y8", fill)
    rt.qmm_i8("w8", "q8", "s8", "y8", ntok)
    rt.synchronize()
    y = rt.read_array("y8")
    assert (y[ntok * rows:] == 3.0).all()
    y = y[:ntok * rows].reshape(ntok, rows).astype(np.float64)
    want, _ = F.qmm_i8(w, ws, q, qs)
    off = np.abs(y - want) - bound(want, kind)
    assert (off <= 0).all(), (np.argwhere(off > 0)[:5], y.flat[off.argmax()], want.flat[off.argmax()])
    return y


@pytest.mark.parametrize("ntok", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 63, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513])
def test_product_at_every_number_of_rows(rt, ntok):
    rng = np.random.default_rng(ntok)
    for rows, cols in ((257, 512), (130, 1000)):
        check_product(rt, *make(rng, rows, cols, ntok))


@pytest.mark.parametrize("cols", [1, 2, 3, 4, 15, 16, 17, 31, 100, 127, 128, 129, 255, 256, 257, 640, 1111, 4096, 5120, 10001])
def test_product_at_every_length(rt, cols):
    rng = np.random.default_rng(cols)
    for rows, ntok in ((1, 1), (33, 6), (300, 40), (129, 130)):
        check_product(rt, *make(rng, rows, cols, ntok), kind=np.float16 if cols in (17, 129, 5120) else np.float32)


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 127, 128, 129, 255, 256, 257, 511, 1001, 5000])
def test_product_at_every_number_of_weight_rows(rt, rows):
    rng = np.random.default_rng(rows)
    for cols, ntok in ((384, 1), (96, 70), (2000, 9), (300, 200)):
        check_product(rt, *make(rng, rows, cols, ntok))


@pytest.mark.parametrize("rows,cols,ntok", [(17408, 5120, 1), (17408, 5120, 4), (5120, 17408, 24), (1024, 5120, 8), (6144, 5120, 64), (151936, 256, 3), (5120, 1000, 700)])
def test_product_on_shapes_of_models(rt, rows, cols, ntok):
    rng = np.random.default_rng(rows)
    w, ws, q, qs = make(rng, rows, cols, ntok)
    check_product(rt, w, ws, q, qs)
    check_product(rt, w, ws, q, qs, kind=np.float16)


@pytest.mark.parametrize("rows,cols,ntok", [(600, 17408, 30), (600, 17408, 40), (600, 17408, 70), (600, 17408, 130), (600, 17408, 256), (300, 20000, 300), (3000, 9000, 600), (1100, 2050, 48),
                                            (1100, 2050, 49), (1100, 2050, 80), (1100, 2050, 81), (20000, 300, 33), (20000, 300, 300), (40000, 130, 257), (256, 256, 4097)])
def test_product_split_by_columns_and_not(rt, rows, cols, ntok):
    """Columns shared by the blocks of a cluster, with memory of their own for the sums and without; tiles that blocks take one after the other."""
    rng = np.random.default_rng(ntok)
    w, ws, q, qs = make(rng, rows, cols, ntok)
    check_product(rt, w, ws, q, qs, kind=np.float16 if ntok in (40, 600) else np.float32)


@pytest.mark.parametrize("ntok", [1, 40])
def test_largest_sums_are_exact(rt, ntok):
    """131071 products of (-128)^2: 2^31 - 2^14, the largest sum there is."""
    rng = np.random.default_rng(1)
    w, _, q, _ = make(rng, 5, 131071, ntok, extreme=True)
    ones = np.ones(5, np.float32), np.ones(ntok, np.float32)
    y = check_product(rt, w, ones[0], q, ones[1])
    assert (y == np.float32(131071 * 16384)).all()


def test_sums_up_to_24_bits_come_back_whole(rt):
    rng = np.random.default_rng(2)
    w, _, q, _ = make(rng, 300, 777, 50)
    y = check_product(rt, w, np.ones(300, np.float32), q, np.ones(50, np.float32))
    assert np.array_equal(y, q.astype(np.int64) @ w.astype(np.int64).T)


def test_a_result_does_not_depend_on_the_rows_beside_it(rt):
    rng = np.random.default_rng(4)
    w, ws, q, qs = make(rng, 700, 2048, 300)
    whole = check_product(rt, w, ws, q, qs)
    for a, b in ((0, 1), (5, 9), (40, 72), (100, 300)):
        assert np.array_equal(check_product(rt, w, ws, q[a:b], qs[a:b]), whole[a:b])


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,ntok", [(200, 1), (333, 20), (513, 150)])
def test_product_onto_what_is_there(rt, rows, ntok, kind):
    rng = np.random.default_rng(rows)
    w, ws, q, qs = make(rng, rows, 400, ntok)
    ws *= np.float32(0.01)
    y0 = rng.standard_normal((ntok, rows)).astype(kind)
    rt.upload_i8("w8", w, ws, 400, rows)
    put_q(rt, "q8", q)
    put(rt, "s8", qs)
    put(rt, "y8", y0)
    rt.qmm_i8("w8", "q8", "s8", "y8", ntok, add=True)
    y = rt.read_array("y8").reshape(ntok, rows).astype(np.float64)
    v, _ = F.qmm_i8(w, ws, q, qs)
    want = y0.astype(np.float64) + v
    # the product's own roundings, then the sum's in fp32, and for fp16 the last one
    limit = 3 * 2.0**-24 * 1.01 * np.abs(v) + 2.0**-24 * 1.01 * np.abs(want) + (2.0**-11 * 1.01 * np.abs(want) + 2.0**-25 if kind is np.float16 else 0)
    assert (np.abs(y - want) <= limit).all()


def test_undefined_scales_make_their_outputs_undefined(rt):
    rng = np.random.default_rng(6)
    for ntok in (5, 80):
        w, ws, q, qs = make(rng, 150, 256, ntok)
        qs[3], ws[17] = np.nan, np.inf
        q[3] = 0
        rt.upload_i8("w8", w, ws, 256, 150)
        put_q(rt, "q8", q)
        put(rt, "s8", qs)
        rt.alloc("y8", ntok * 150)
        rt.qmm_i8("w8", "q8", "s8", "y8", ntok)
        y = rt.read_array("y8").reshape(ntok, 150)
        assert np.isnan(y[3]).all() and not np.isfinite(y[:, 17]).any()
        rest = np.delete(np.delete(y, 3, 0), 17, 1)
        assert np.isfinite(rest).all()


@pytest.mark.parametrize("ntok", [1, 30, 200])
def test_bound_tensors_of_any_pitch(rt, ntok):
    import torch

    rng = np.random.default_rng(ntok)
    w, ws, q, qs = make(rng, 140, 203, ntok)
    full = np.full((140, 272), 55, np.int8)  # what lies behind the columns is not zero
    full[:, :203] = w
    wt, st = torch.from_numpy(full).cuda(), torch.from_numpy(ws).cuda()
    rt.bind_i8("w8", wt.data_ptr(), st.data_ptr(), 203, 140, pitch=272)
    info = rt.tensor_info("w8")
    assert info[1] == 24 and info[2:5] == (140, 203, 272)
    check_product(rt, w, ws, q, qs, bind=True)
    rt.free("w8")
    assert not rt.has("w8")


def test_tensors_beyond_4_gb(rt):
    """Offsets that pass 32 bits: the last rows of a 4.6 GB tensor."""
    import torch

    rows, cols = 281000, 16384
    w = torch.zeros((rows, cols), dtype=torch.int8, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    ends = [0, 131071, 131072, 262143, 262144, 270000, rows - 1]
    w[ends] = torch.randint(-128, 128, (len(ends), cols), generator=gen, device="cuda", dtype=torch.int8)
    ws = torch.rand(rows, generator=gen, device="cuda") + 0.5
    torch.cuda.synchronize()
    rng = np.random.default_rng(0)
    for ntok in (1, 9, 140):
        q = rng.integers(-128, 128, (ntok, cols), dtype=np.int8)
        qs = rng.uniform(0.5, 1.5, ntok).astype(np.float32)
        rt.bind_i8("w8", w.data_ptr(), ws.data_ptr(), cols, rows)
        put_q(rt, "q8", q)
        put(rt, "s8", qs)
        y = torch.empty((ntok, rows), device="cuda")
        rt.bind("y8", y.data_ptr(), y.numel())
        rt.qmm_i8("w8", "q8", "s8", "y8", ntok)
        rt.synchronize()
        want, _ = F.qmm_i8(w[ends].cpu().numpy(), ws[ends].cpu().numpy(), q, qs)
        assert (np.abs(y[:, ends].cpu().numpy() - want) <= bound(want, np.float32)).all()
        assert int((y != 0).sum()) == int((y[:, ends] != 0).sum())
        rt.release("y8")
    rt.free("w8")


@pytest.mark.parametrize("t", [T.F32, T.F16, T.Q8_0, T.Q4_K, T.Q6_K, T.Q3_K, T.IQ3_S, T.IQ4_NL], ids=lambda t: t.name)
def test_conversion_of_gguf_tensors(rt, t):
    from vinf_3080ti_b200.synth import synthetic_blocks

    rng = np.random.default_rng(int(t))
    rows, cols = (77, 520) if t in (T.F32, T.F16) else (77, 512)
    rt.upload("from", synthetic_blocks(t, rows, cols, rng), int(t), cols, rows)
    rt.alloc("full", rows * cols)
    rt.dequantize("from", "full")
    want_q, want_s, _ = F.rows_i8(rt.read_array("full").reshape(rows, cols))
    rt.convert_i8("from", "to")
    # read back through products with one-hot activations
    info = rt.tensor_info("to")
    assert info[1:5] == (24, rows, cols, F.pitch(cols))
    q = np.zeros((cols, cols), np.int8)
    q[np.arange(cols), np.arange(cols)] = 1
    put_q(rt, "q8", q, junk=0)
    put(rt, "s8", np.ones(cols, np.float32))
    rt.alloc("y8", cols * rows)
    rt.qmm_i8("to", "q8", "s8", "y8", cols)
    y = rt.read_array("y8").reshape(cols, rows).T
    assert np.array_equal(y, want_q.astype(np.float32) * want_s[:, None])
    rt.convert_i8("from", "from")  # in its own place
    assert rt.tensor_info("from")[1] == 24


def test_conversion_in_parts(rt):
    """More than 16 Mi elements: several parts, the last one shorter."""
    rng = np.random.default_rng(0)
    rows, cols = 4133, 8192
    w = rng.standard_normal((rows, cols)).astype(np.float32)
    rt.upload("from", w, int(T.F32), cols, rows)
    rt.convert_i8("from", "to")
    want_q, want_s, _ = F.rows_i8(w)
    q = rng.integers(-128, 128, (2, cols), dtype=np.int8)
    put_q(rt, "q8", q)
    put(rt, "s8", np.ones(2, np.float32))
    rt.alloc("y8", 2 * rows)
    rt.qmm_i8("to", "q8", "s8", "y8", 2)
    want, _ = F.qmm_i8(want_q, want_s, q, np.ones(2, np.float32))
    assert (np.abs(rt.read_array("y8").reshape(2, rows) - want) <= bound(want, np.float32)).all()
    rt.free("from")
    rt.free("to")


# ---- refusals ---------------------------------------------------------------------------------------------------------


def test_refusals(rt):
    rt.upload_i8("w8", np.zeros((4, 40), np.int8), np.ones(4, np.float32), 40, 4)
    rt.upload("gguf", np.zeros(4 * 64, np.float32), int(T.F32), 64, 4)
    for name, n, elem in (("x", 120, 4), ("h", 120, 2), ("q", 144, 1), ("q1", 143, 1), ("s", 3, 4), ("s2", 2, 4), ("y", 12, 4), ("y11", 11, 4), ("g", 40, 4)):
        rt.alloc(name, n, elem)
    ok = dict(x="x", q="q", scales="s", cols=40, ntok=3)

    def rows(**kw):
        a = {**ok, **kw}
        rt.rows_i8(a.pop("x"), a.pop("q"), a.pop("scales"), a.pop("cols"), a.pop("ntok"), **a)

    rows()
    for error, kw in ((ValueError, {"ntok": 0}), (ValueError, {"ntok": -1}), (ValueError, {"ntok": 4}), (ValueError, {"cols": 0}), (ValueError, {"cols": 131072}),
                      (ValueError, {"q": "q1"}), (TypeError, {"q": "x"}), (TypeError, {"x": "q"}), (TypeError, {"scales": "h"}), (ValueError, {"scales": "s2"}),
                      (KeyError, {"x": "none"}), (KeyError, {"norm": "none"}), (ValueError, {"norm": "s"}), (ValueError, {"norm": "g", "eps": -1.0}),
                      (ValueError, {"norm": "g", "eps": float("nan")}), (TypeError, {"residual": "h"}), (TypeError, {"silu_mul": "h"}), (ValueError, {"total": "x"}),
                      (TypeError, {"residual": "x", "total": "h"}), (ValueError, {"residual": "x", "silu_mul": "x"}), (ValueError, {"norm": "gguf"}),
                      (ValueError, {"norm": "w8"}), (ValueError, {"silu_mul": "s"})):
        with pytest.raises(error):
            rows(**kw)
    rt.qmm_i8("w8", "q", "s", "y", 3)
    for error, a in ((ValueError, ("w8", "q", "s", "y", 0)), (ValueError, ("w8", "q1", "s", "y", 3)), (ValueError, ("w8", "q", "s2", "y", 3)),
                     (ValueError, ("w8", "q", "s", "y11", 3)), (ValueError, ("gguf", "q", "s", "y", 3)), (KeyError, ("none", "q", "s", "y", 3)),
                     (TypeError, ("w8", "x", "s", "y", 3)), (TypeError, ("w8", "q", "s", "q", 3)), (ValueError, ("w8", "q", "s", "y", 2**31 - 1))):
        with pytest.raises(error):
            rt.qmm_i8(*a)
    # the matvecs of GGUF blocks refuse these tensors
    for call in (lambda: rt.qmv("w8", "x", "y", 1), lambda: rt.qmv_argmax("w8", "x", None, 1), lambda: rt.qmv_fused("w8", "x", "y", 1),
                 lambda: rt.qmv_group(["w8"], "x", ["y"], 1), lambda: rt.matvec("w8", np.zeros(40, np.float32)), lambda: rt.dequantize("w8", "x"),
                 lambda: rt.convert_i8("w8", "other"), lambda: rt.set_argmax_row_base("w8", 1), lambda: rt.qmv_push("w8", "x", "y", 1, -1, 0, 4, 0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        rt.qmv("gguf", "q", "y", 1)
    for a in (("n", np.zeros(7, np.int8), np.ones(2, np.float32), 4, 2), ("n", np.zeros(8, np.int8), np.ones(1, np.float32), 4, 2), ("n", np.zeros(0, np.int8), np.ones(2, np.float32), 0, 2),
              ("n", np.zeros(131072, np.int8), np.ones(1, np.float32), 131072, 1)):
        with pytest.raises(ValueError):
            rt.upload_i8(*a)
    addr = rt.buffer_ptr("x")[0]
    for a, kw in (((addr + 8, addr, 16, 1), {}), ((addr, addr + 2, 16, 1), {}), ((0, addr, 16, 1), {}), ((addr, 0, 16, 1), {}), ((addr, addr, 16, 1), {"pitch": 8}),
                  ((addr, addr, 16, 1), {"pitch": 24}), ((addr, addr, 17, 1), {"pitch": 16}), ((addr, addr, 16, 0), {}), ((addr, addr, 16, 1), {"pitch": -16})):
        with pytest.raises(ValueError):
            rt.bind_i8("n", *a, **kw)
    with pytest.raises(KeyError):
        rt.convert_i8("none", "n")
    rt.upload("odd", np.zeros(9, np.float32), int(T.F32), 3, 3)
    with pytest.raises(ValueError):
        rt.convert_i8("odd", "n")
    with pytest.raises(ValueError):
        rt.alloc("n", 4, 3)
    assert not rt.has("n")
    rt.capture_begin()
    try:
        for call in (lambda: rt.convert_i8("gguf", "n"), lambda: rt.upload_i8("n", np.zeros(4, np.int8), np.ones(1, np.float32), 4, 1)):
            with pytest.raises(ValueError):
                call()
        rt.qmm_i8("w8", "q", "s", "y", 3)
    finally:
        rt.graph_destroy(rt.capture_end())
    rt.synchronize()


def test_what_is_written_has_a_buffer_of_its_own(rt):
    rt.upload_i8("w8", np.zeros((2, 4), np.int8), np.ones(2, np.float32), 4, 2)
    for name, n, elem in (("x", 8, 4), ("r", 8, 4), ("q", 32, 1), ("s", 4, 4), ("g", 4, 4), ("y", 4, 4)):
        rt.alloc(name, n, elem)
    for kw in (dict(x="s", scales="s", ntok=1), dict(silu_mul="s", ntok=1), dict(norm="s"), dict(residual="s", total="r", ntok=1), dict(residual="r", total="s", ntok=1),
               dict(residual="g", norm="g", ntok=1)):
        a = {**dict(x="x", q="q", scales="s", cols=4, ntok=2), **kw}
        with pytest.raises(ValueError, match="of their own"):
            rt.rows_i8(a.pop("x"), a.pop("q"), a.pop("scales"), a.pop("cols"), a.pop("ntok"), **a)
    with pytest.raises(ValueError, match="of their own"):
        rt.qmm_i8("w8", "q", "s", "s", 2)
    rt.rows_i8("x", "q", "s", 4, 2, residual="r", total="x", norm="g")
    rt.qmm_i8("w8", "q", "s", "y", 2)
    rt.synchronize()


def test_more_rows_than_an_integer_counts_by_tiles_are_refused(rt):
    rt.alloc("x", 4)
    at = rt.buffer_ptr("x")[0]
    for rows in (2**30 + 1, 2**31 - 1):
        with pytest.raises(ValueError, match="at most"):
            rt.bind_i8("n", at, at, 16, rows)
    rt.upload_i8("w8", np.zeros((2, 4), np.int8), np.ones(2, np.float32), 4, 2)
    rt.alloc("q", 32, 1)
    for ntok in (2**30 + 1, 2**31 - 1):
        with pytest.raises(ValueError, match="ntok"):
            rt.qmm_i8("w8", "q", "x", "x", ntok)


def test_bytes_are_written_copied_and_read(rt):
    data = np.arange(-100, 100, dtype=np.int8)
    rt.alloc("b", 200, 1)
    rt.alloc("c", 50, 1)
    rt.write("b", data)
    rt.copy("c", 10, "b", 30, 20)
    assert rt.buffer_elem("b") == 1
    assert np.array_equal(rt.read_array("b", 5, 7), data[7:12])
    assert np.array_equal(rt.read_array("c"), np.concatenate([np.zeros(10, np.int8), data[30:50], np.zeros(20, np.int8)]))
    rt.zero_range("b", 3, 4)
    assert np.array_equal(rt.read_array("b", 10), np.where((np.arange(10) >= 3) & (np.arange(10) < 7), 0, data[:10]))
