"""Passes in 8-bit floating point on the GPU against their formulas in 64 bits (tests/f8_formulas.py).

Tolerances, in units u = 2^-24 (a rounding of fp32 is off by at most one u of the value).

Values: without norm or gate they are exact, so scales and e4m3 values are equal to the formula's.  A norm: the sum of squares is off by 1 for each square and 1
for each addition on the way (at most 64 of a thread's, 10 over warps), the mean and eps by 2, half of which the root keeps, and 2 for root and reciprocal; two products:
less than 44.  A gate: the exponential 4 (2 ulp), its square 9, of which 1 / (1 + h^2) keeps half, the sum, the division, three products and the exponential in two of them: less than 20;
in a norm's mean they count once more.  The scale's division 1 and the quotient's 1.
The scale is within that of max |n| / 448, and the e4m3 value is a nearest one of some value within that of n / scale.

Products: e4m3 times e4m3 is exact.  A block's 128 products are added in the tensor core in fp32, with cut-off digits: 2 u for each, of the sum of their magnitudes; the
scales' product, its product with the sum and the addition over blocks 1 each.  fp16 outputs one rounding more of 2^-11 (2^-25 among subnormals).  Where all sums are small whole
numbers and scales powers of two nothing is rounded: then results are equal.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests import f8_formulas as F
from vinf_3080ti_b200.gguf_types import GGUFTensorType as T
from vinf_3080ti_b200.gguf_types import row_bytes

pytestmark = pytest.mark.gpu

NORM, GATE = 44 * F.U, 20 * F.U


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
    n_scales = F.blocks(cols) * F.scale_pitch(ntok)
    put(rt, "s", np.full(n_scales + 1, 7.0, np.float32))
    if x2 is not None:
        put(rt, "x2", x2)
    if residual is not None:
        put(rt, "r", residual)
        if total == "t":
            put(rt, "t", np.zeros_like(x))
    if norm is not None:
        put(rt, "g", norm)
    rt.rows_f8("x", "q", "s", cols, ntok, residual=None if residual is None else "r", total=total, norm=None if norm is None else "g", eps=eps,
               silu_mul=None if x2 is None else "x2")
    rt.synchronize()
    q = rt.read_array("q").view(np.uint8)
    assert (q[ntok * F.pitch(cols):] == 99).all()  # nothing behind the last row
    q = q[:ntok * F.pitch(cols)].reshape(ntok, F.pitch(cols))
    assert (q[:, cols:] == 0).all()
    s = rt.read_array("s")
    assert s[n_scales] == 7.0
    s = s[:n_scales].reshape(F.blocks(cols), F.scale_pitch(ntok))
    assert (s[:, ntok:] == 7.0).all()
    got_total = None if residual is None else rt.read_array(total or "r").reshape(ntok, cols)
    return q[:, :cols], s[:, :ntok], got_total


def check_rows(rt, x, total=None, **kw):
    q, s, t = run_rows(rt, x, total=total, **kw)
    n, want_t = F.values(x, **kw)
    if want_t is not None:
        assert np.array_equal(t, want_t, equal_nan=True)
    gate, norm = kw.get("x2") is not None, kw.get("norm") is not None
    off = (2 * GATE if norm else GATE) * gate + NORM * norm
    want_s = F.scales_of(n)
    bad = np.isnan(want_s)
    assert np.array_equal(np.isnan(s), bad)
    got, spread = F.CODES[q], F.spread_scales(s.astype(np.float64), x.shape[1])
    assert not np.isnan(got).any() and (got[np.isnan(spread)] == 0).all()
    if off == 0:
        assert np.array_equal(s, want_s.astype(np.float32), equal_nan=True)
        some = spread > 0
        want = np.zeros(q.shape, np.uint8)
        want[some] = F.encode((n[some] / spread[some]).astype(np.float32))
        assert np.array_equal(q & np.where(got == 0, 127, 255), want & np.where(F.CODES[want] == 0, 127, 255))
        return
    fine = ~bad
    assert (np.abs(s - want_s)[fine] <= (off + F.U) * 1.01 * want_s[fine] + 2.0**-149).all()
    some = (spread > 2.0**-120) & np.isfinite(n)
    t = n[some] / spread[some]  # (by the scale that is stored)
    miss = np.abs(got[some] - t) - F.step(t * (1 + off)) / 2 - np.abs(t) * (off + 2 * F.U) * 1.01
    # the largest may end a hair beyond 448
    miss = np.where((np.abs(t) > 448) & (np.abs(got[some]) == 448), np.abs(t) / 448 - 1 - (off + 2 * F.U) * 1.01, miss)
    assert (miss <= 0).all(), (miss.max(), t[miss.argmax()], got[some][miss.argmax()])


COLS = [1, 2, 7, 8, 9, 15, 16, 17, 64, 127, 128, 129, 255, 256, 257, 1000, 2047, 4099, 5120, 8200, 17408]


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("cols", COLS)
def test_rows_of_every_length(rt, cols, kind):
    rng = np.random.default_rng(cols)
    for ntok in (1, 3, 4, 5):
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


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("cols", [16384, 16392, 24576, 24577, 32768, 32769, 40001, 65536, 131072, 200003])
def test_long_rows(rt, cols, kind):
    rng = np.random.default_rng(cols)
    x, res = rng.standard_normal((2, 2, cols)).astype(kind)
    g = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    check_rows(rt, x)
    check_rows(rt, x, residual=res, norm=g)
    check_rows(rt, x, residual=res, norm=g, total="t")
    check_rows(rt, x, x2=res)
    check_rows(rt, x, x2=res, norm=g)


@pytest.mark.parametrize("ntok,cols", [(700, 520), (3000, 64), (149, 5120), (301, 5121), (1025, 1000), (170, 12288)])
def test_many_rows(rt, ntok, cols):
    rng = np.random.default_rng(ntok)
    for kind in (np.float32, np.float16):
        x, res = rng.standard_normal((2, ntok, cols)).astype(kind)
        check_rows(rt, x)
        check_rows(rt, x, x2=res)
        check_rows(rt, x, residual=res, norm=rng.uniform(0.5, 1.5, cols).astype(np.float32), total="t")


def test_halves_go_to_even(rt):
    """Scale 1; halves between all e4m3 values, and fp32 values to either side of them."""
    half = ((F.CODES[:126] + F.CODES[1:127]) / 2).astype(np.float32)
    for row in (half, np.nextafter(half, np.float32(1e9)), np.nextafter(half, np.float32(-1)), -half):
        x = np.concatenate([row, [448, -448]]).astype(np.float32)[None]
        q, s, _ = run_rows(rt, x)
        assert s.tolist() == [[1.0]]
        assert np.array_equal(q, F.encode(x))


def test_zero_tiny_and_huge_rows(rt):
    x = np.zeros((9, 300), np.float32)
    x[1, 5] = 1e-44       # the scale rounds to a subnormal or to zero
    x[2] = 1e-38
    x[3, ::2] = 3e38      # squares beyond fp32
    x[4, 1] = -3.4e38
    x[5] = np.float32(1e-30)
    x[6, 0], x[6, 1] = 1.0, 1e-30
    x[7] = -5.0
    x[8, 129] = 448.0     # blocks of zeros beside one that is not
    check_rows(rt, x)
    check_rows(rt, x[3:], norm=np.ones(300, np.float32), eps=1e-6)
    check_rows(rt, x[[1, 2, 5, 6]], norm=np.ones(300, np.float32), eps=1e-6)
    q, s, _ = run_rows(rt, np.zeros((2, 300), np.float32), norm=np.ones(300, np.float32))
    assert not q.any() and not s.any()
    q, s, _ = run_rows(rt, np.zeros((2, 300), np.float32), norm=np.ones(300, np.float32), eps=0.0)
    assert not q.any() and np.isnan(s).all()  # 0 / 0


@pytest.mark.parametrize("cols", [64, 67, 1536])
def test_norms_of_values_at_the_ends_of_fp32(rt, cols):
    """Sums of squares that fp32 does not hold, and weights that bring the products back."""
    rng = np.random.default_rng(cols)
    g = rng.uniform(0.5, 1.5, cols)
    x = rng.standard_normal((40, cols))
    for size, weight in ((1e-35, 1e20), (1e-30, 1.0), (8e37, 1e-20), (8e37, 1e-8), (3e37, 1.0), (1e20, 1.0)):
        check_rows(rt, (x.clip(-4, 4) * size).astype(np.float32), norm=(g * weight).astype(np.float32), eps=0.0)


def test_gated_values_far_from_zero(rt):
    """Large negative x, whose silu is all but nothing, beside ordinary ones and beside large x2."""
    rng = np.random.default_rng(13)
    x = np.concatenate([np.linspace(-120, 120, 601), [-88.5, -87.0, -103.0, -150.0, 1e4, -1e4]]).astype(np.float32)
    x = np.tile(x, (6, 1))
    x2 = rng.standard_normal(x.shape).astype(np.float32)
    x[1] = np.minimum(x[1], -79)
    x[2] = np.minimum(x[2], -95)
    x2[2] *= np.float32(1e25)
    x2[3, ::7] = 1e20
    x2[5, ::5] = 1e30
    check_rows(rt, x, x2=x2)
    check_rows(rt, x[[0, 3, 5]], x2=x2[[0, 3, 5]], norm=np.ones(x.shape[1], np.float32))


def test_undefined_blocks_have_an_undefined_scale_and_leave_the_others_alone(rt):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 333)).astype(np.float32)
    x[1, 7], x[2, 332], x[4, 0] = np.nan, np.inf, -np.inf
    g = np.ones(333, np.float32)
    check_rows(rt, x)
    assert np.argwhere(np.isnan(rt.read_array("s")[:24].reshape(3, 8)[:, :6])).tolist() == [[0, 1], [0, 4], [2, 2]]
    check_rows(rt, x, residual=np.ones_like(x))
    for kw in ({"norm": g}, {"residual": np.ones_like(x), "norm": g}):
        # the root mean square of a row with a NaN is undefined, of one with an infinite value infinite, which leaves zeros of the others
        q, s, _ = run_rows(rt, x, **kw)
        assert np.argwhere(np.isnan(s)).tolist() == [[0, 1], [0, 4], [1, 1], [2, 1], [2, 2]]
        assert not q[[1, 2, 4]].any() and q[[0, 3, 5]].any(1).all() and s[1, 4] == 0 and s[0, 2] == 0
        check_rows(rt, x, **kw)
    # fp16 sums beyond 65504 are infinite
    half = np.full((1, 40), 60000, np.float16)
    check_rows(rt, half, residual=half)


def test_norm_weights_may_be_a_tensor(rt):
    rng = np.random.default_rng(8)
    g = rng.uniform(0.5, 1.5, 128).astype(np.float32)
    x = rng.standard_normal((3, 128)).astype(np.float32)
    rt.upload("gain", g, int(T.F32), 128, 1)
    want_q, want_s, _ = run_rows(rt, x, norm=g)
    rt.rows_f8("x", "q", "s", 128, 3, norm="gain")
    assert np.array_equal(rt.read_array("q").view(np.uint8)[:384].reshape(3, 128), want_q) and np.array_equal(rt.read_array("s")[:4].reshape(1, 4)[:, :3], want_s)


# ---- the product ------------------------------------------------------------------------------------------------------


def make(rng, rows, cols, ntok, whole=False):
    if whole:  # small whole numbers, scales that are powers of two
        small = F.encode(np.arange(-3, 4))
        w, q = (small[rng.integers(0, 7, (n, cols))] for n in (rows, ntok))
        ws, qs = (np.exp2(rng.integers(-1, 2, shape)).astype(np.float32) for shape in ((F.blocks(rows), F.blocks(cols)), (F.blocks(cols), ntok)))
    else:
        w, q = (F.encode(rng.standard_normal((n, cols)) * 100) for n in (rows, ntok))
        ws, qs = (rng.uniform(1e-4, 1e-2, shape).astype(np.float32) for shape in ((F.blocks(rows), F.blocks(cols)), (F.blocks(cols), ntok)))
    return w, ws, q, qs


def put_rows(rt, q, qs, junk=0x7F):
    """Rows at their pitch; what lies behind a row's columns, and behind a block's scales, is not a number."""
    full = np.full((q.shape[0], F.pitch(q.shape[1])), junk, np.uint8)
    full[:, :q.shape[1]] = q
    put(rt, "q8", full.view(np.int8))
    scales = np.full((qs.shape[0], F.scale_pitch(qs.shape[1])), np.nan, np.float32)
    scales[:, :qs.shape[1]] = qs
    put(rt, "s8", scales)


def bound(most, want, cols, kind):
    b = most * (2 * F.BLOCK + 3 + F.blocks(cols)) * F.U * 1.01 + 2.0**-149
    return b + (np.abs(want) + b) * 2.0**-11 + 2.0**-25 if kind is np.float16 else b


def check_product(rt, w, ws, q, qs, kind=np.float32, whole=False, upload=True, before=None):
    (rows, cols), ntok = w.shape, q.shape[0]
    if upload:
        rt.upload_f8("w8", w, ws, cols, rows)
    put_rows(rt, q, qs)
    fill = np.full(ntok * rows + 5, 3.0, kind)
    if before is not None:
        fill[:ntok * rows] = before.reshape(-1)
    put(rt, "y8", fill)
    rt.qmm_f8("w8", "q8", "s8", "y8", ntok, add=before is not None)
    rt.synchronize()
    y = rt.read_array("y8")
    assert (y[ntok * rows:] == 3.0).all()
    y = y[:ntok * rows].reshape(ntok, rows).astype(np.float64)
    want, most = F.qmm(w, ws, q, qs)
    if before is not None:
        want, most = want + before, most + np.abs(before)
    if whole:
        assert np.array_equal(y, want.astype(kind)), np.argwhere(y != want)[:5]
    else:
        off = np.abs(y - want) - bound(most, want, cols, kind)
        assert (off <= 0).all(), (np.argwhere(off > 0)[:5], y.flat[off.argmax()], want.flat[off.argmax()])
    return y


NTOK = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 384, 385, 513]


@pytest.mark.parametrize("ntok", NTOK)
def test_product_at_every_number_of_rows(rt, ntok):
    rng = np.random.default_rng(ntok)
    for rows, cols in ((257, 512), (130, 1000)):
        check_product(rt, *make(rng, rows, cols, ntok, whole=True), whole=True)
        check_product(rt, *make(rng, rows, cols, ntok))


@pytest.mark.parametrize("cols", [1, 2, 15, 16, 17, 100, 127, 128, 129, 255, 256, 257, 640, 1111, 4096, 5120, 10001])
def test_product_at_every_length(rt, cols):
    rng = np.random.default_rng(cols)
    for rows, ntok in ((1, 1), (33, 6), (300, 40), (129, 130)):
        kind = np.float16 if cols in (17, 129, 5120) else np.float32
        check_product(rt, *make(rng, rows, cols, ntok), kind=kind)
        if kind is np.float32:
            check_product(rt, *make(rng, rows, cols, ntok, whole=True), whole=True)


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 127, 128, 129, 255, 256, 257, 511, 1001, 5000])
def test_product_at_every_number_of_weight_rows(rt, rows):
    rng = np.random.default_rng(rows)
    for cols, ntok in ((384, 1), (96, 70), (2000, 9), (300, 200)):
        check_product(rt, *make(rng, rows, cols, ntok, whole=True), whole=True)
        check_product(rt, *make(rng, rows, cols, ntok), kind=np.float16)


@pytest.mark.parametrize("rows,cols,ntok", [(17408, 5120, 1), (17408, 5120, 4), (5120, 17408, 24), (1024, 5120, 8), (6144, 5120, 64), (151936, 256, 3), (5120, 1000, 700), (1024, 5120, 300)])
def test_product_on_shapes_of_models(rt, rows, cols, ntok):
    rng = np.random.default_rng(rows)
    w, ws, q, qs = make(rng, rows, cols, ntok, whole=cols <= 5120)
    check_product(rt, w, ws, q, qs, whole=cols <= 5120)
    check_product(rt, w, ws, q, qs, kind=np.float16, upload=False)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols,ntok", [(40000, 200, 3), (40000, 200, 17), (40000, 200, 40), (40000, 200, 100), (30001, 136, 120), (40000, 200, 300), (20000, 130, 700), (20004, 300, 130)])
def test_product_of_more_tiles_than_fit_at_once(rt, rows, cols, ntok, kind):
    """Blocks take several tiles, one after the other; a tile's outputs are still on their way when the next one's are made."""
    rng = np.random.default_rng(rows + ntok)
    w, ws, q, qs = make(rng, rows, cols, ntok, whole=True)
    ws[:] = 1.0
    qs[:] = 1.0 / 16
    check_product(rt, w, ws, q, qs, kind=kind, whole=True)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols,ntok", [(5120, 8192, 256), (4993, 8200, 200), (4994, 8100, 129), (4996, 8300, 255), (5900, 14300, 140), (3300, 4400, 250), (2049, 5120, 500), (129, 17408, 257)])
def test_product_of_wide_tiles_whose_columns_are_shared(rt, rows, cols, ntok, kind):
    """Tiles of 256 x 256 by two and three parts of the columns, and sizes beside those that have them."""
    rng = np.random.default_rng(rows + cols)
    check_product(rt, *make(rng, rows, cols, ntok, whole=cols <= 5120), kind=kind, whole=cols <= 5120)
    check_product(rt, *make(rng, rows, cols, ntok), kind=kind, before=rng.standard_normal((ntok, rows)).astype(kind))


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols,ntok", [(1, 1, 1), (257, 300, 4), (1000, 2000, 33), (300, 5120, 1), (129, 129, 128), (257, 512, 200), (999, 700, 300)])
def test_product_onto_what_is_there(rt, rows, cols, ntok, kind):
    rng = np.random.default_rng(rows)
    before = rng.standard_normal((ntok, rows)).astype(kind)
    check_product(rt, *make(rng, rows, cols, ntok), kind=kind, before=before)


def test_undefined_scales_and_values_stay_in_their_rows(rt):
    """A NaN scale of a row, a NaN byte of a row, a NaN scale of a block of weights: what they multiply is undefined, nothing else is."""
    rng = np.random.default_rng(6)
    for ntok in (3, 40, 140):
        w, ws, q, qs = make(rng, 300, 400, ntok)
        qs[1, 1] = np.nan
        q[2, 399] = 0x7F
        ws[2, 3] = np.nan
        rt.upload_f8("w8", w, ws, 400, 300)
        put_rows(rt, q, qs)
        rt.alloc("y8", ntok * 300)
        rt.qmm_f8("w8", "q8", "s8", "y8", ntok)
        y = rt.read_array("y8").reshape(ntok, 300)
        want = np.zeros((ntok, 300), bool)
        want[1:3] = True
        want[:, 256:] = True
        assert np.array_equal(np.isnan(y), want)


@pytest.mark.parametrize("cols,pitch,ntok", [(100, 112, 3), (100, 256, 3), (128, 144, 40), (1000, 1024, 140)])
def test_bound_weights_with_a_pitch(rt, cols, pitch, ntok):
    """Rows further apart than they are long, with bytes behind them that are not numbers."""
    import torch

    rng = np.random.default_rng(pitch)
    w, ws, q, qs = make(rng, 200, cols, ntok, whole=True)
    full = np.full((200, pitch), 0x7F, np.uint8)
    full[:, :cols] = w
    dev, scales = torch.from_numpy(full).cuda(), torch.from_numpy(ws).cuda()
    torch.cuda.synchronize()
    rt.bind_f8("w8", dev.data_ptr(), scales.data_ptr(), cols, 200, pitch=0 if pitch == F.pitch(cols) else pitch)
    assert rt.tensor_info("w8")[1:5] == (128, 200, cols, pitch)
    check_product(rt, w, ws, q, qs, whole=True, upload=False)
    rt.synchronize()
    rt.free("w8")


@pytest.mark.parametrize("kind,rows,cols", [(T.Q4_K, 300, 512), (T.Q6_K, 129, 256), (T.F32, 131, 136), (T.F16, 7, 24), (T.Q8_0, 260, 1056)])
def test_conversion_of_gguf_tensors(rt, kind, rows, cols):
    from vinf_3080ti_b200.synth import synthetic_blocks

    rng = np.random.default_rng(rows)
    if kind in (T.F32, T.F16):
        raw = rng.standard_normal(rows * cols).astype(np.float32 if kind == T.F32 else np.float16)
    else:
        raw = synthetic_blocks(kind, rows, cols, rng)
    assert np.ascontiguousarray(raw).nbytes == rows * row_bytes(kind, cols)
    rt.upload("g", raw, int(kind), cols, rows)
    rt.alloc("values", rows * cols)
    rt.dequantize("g", "values")
    w = rt.read_array("values").reshape(rows, cols).astype(np.float64)
    rt.convert_f8("g", "g8")
    scales = np.empty((F.blocks(rows), F.blocks(cols)), np.float32)
    want = np.empty((rows, cols), np.uint8)
    for i in range(F.blocks(rows)):
        for j in range(F.blocks(cols)):
            at = np.s_[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128]
            scales[i, j] = np.abs(w[at]).max() / 448
            want[at] = F.encode((w[at] / np.float64(scales[i, j])).astype(np.float32)) if scales[i, j] > 0 else 0
    addr, type_, r, c, pitch, nbytes, _ = rt.tensor_info("g8")
    assert (type_, r, c, pitch) == (128, rows, cols, F.pitch(cols))
    at = (rows * pitch + 255) // 256 * 256
    rt.bind("raw", addr, at + scales.nbytes, 1)
    raw = rt.read_array("raw").view(np.uint8)
    assert np.array_equal(raw[at:].view(np.float32).reshape(scales.shape), scales)
    got = raw[:rows * pitch].reshape(rows, pitch)
    assert (got[:, cols:] == 0).all()
    assert np.array_equal(got[:, :cols] & np.where(F.CODES[want] == 0, 127, 255), want & np.where(F.CODES[want] == 0, 127, 255))
    rt.release("raw")


# ---- refusals ---------------------------------------------------------------------------------------------------------


def test_refusals(rt):
    rng = np.random.default_rng(1)
    w, ws, q, qs = make(rng, 20, 40, 3)
    for bad in (dict(cols=0), dict(rows=0), dict(cols=-1), dict(cols=(1 << 20) + 1), dict(data=w[:-1]), dict(scales=ws[:0]), dict(scales=np.ones(2, np.float32))):
        with pytest.raises(ValueError):
            rt.upload_f8(**{**dict(name="w8", data=w, scales=ws, cols=40, rows=20), **bad})
    rt.upload_f8("w8", w, ws, 40, 20)
    put_rows(rt, q, qs)
    rt.alloc("y8", 60)
    rt.qmm_f8("w8", "q8", "s8", "y8", 3)
    for call, error in ((lambda: rt.qmm_f8("w8", "q8", "s8", "y8", 0), ValueError), (lambda: rt.qmm_f8("w8", "q8", "s8", "y8", 4), ValueError),
                        (lambda: rt.qmm_f8("w8", "q8", "s8", "y8", 5), ValueError), (lambda: rt.qmm_f8("nothing", "q8", "s8", "y8", 3), KeyError),
                        (lambda: rt.qmm_f8("w8", "s8", "q8", "y8", 3), TypeError), (lambda: rt.qmm_f8("w8", "q8", "s8", "q8", 3), TypeError),
                        (lambda: rt.qmm_f8("w8", "q8", "s8", "s8", 1), ValueError), (lambda: rt.qmm_f8("w8", "q8", "y8", "y8", 1), ValueError),
                        (lambda: rt.qmm_i8("w8", "q8", "s8", "y8", 3), ValueError), (lambda: rt.qmv("w8", "s8", "y8", 1), ValueError),
                        (lambda: rt.matvec("w8", np.zeros(40, np.float32)), ValueError), (lambda: rt.dequantize("w8", "y8"), ValueError), (lambda: rt.convert_f8("w8", "w9"), ValueError),
                        (lambda: rt.convert_i8("w8", "w9"), ValueError), (lambda: rt.qmv_argmax("w8", "s8", None, 1), ValueError),
                        (lambda: rt.bind_f8("w9", 8, 16, 1, 1), ValueError), (lambda: rt.bind_f8("w9", 16, 2, 1, 1), ValueError), (lambda: rt.bind_f8("w9", 16, 16, 20, 1, pitch=16), ValueError),
                        (lambda: rt.bind_f8("w9", 16, 16, 20, 1, pitch=40), ValueError)):
        with pytest.raises(error):
            call()
    rt.upload_i8("wi", np.zeros((20, 40), np.int8), np.ones(20, np.float32), 40, 20)
    with pytest.raises(ValueError, match="8-bit integer rows"):
        rt.qmm_f8("wi", "q8", "s8", "y8", 3)
    put(rt, "x", np.ones((3, 40), np.float32))
    put(rt, "h", np.ones((3, 40), np.float16))
    rt.alloc("q", 3 * 48, 1)
    rt.alloc("s", 4)
    ok = dict(x="x", q="q", scales="s", cols=40, ntok=3)
    rt.rows_f8(**ok)
    for bad, error in ((dict(ntok=0), ValueError), (dict(ntok=4), ValueError), (dict(cols=0), ValueError), (dict(cols=(1 << 20) + 1), ValueError), (dict(x="q"), TypeError), (dict(q="x"), TypeError),
                       (dict(x="h", residual="x"), TypeError), (dict(residual="x", silu_mul="x"), ValueError), (dict(total="x"), ValueError), (dict(norm="s"), ValueError),
                       (dict(norm="x", eps=-1.0), ValueError), (dict(norm="x", eps=float("nan")), ValueError), (dict(scales="h"), TypeError), (dict(scales="x", residual="x"), ValueError)):
        with pytest.raises(error):
            rt.rows_f8(**{**ok, **bad})
    rt.alloc("short", 3)
    with pytest.raises(ValueError):  # the scales' rows are rounded up to 4
        rt.rows_f8(**{**ok, "scales": "short"})
