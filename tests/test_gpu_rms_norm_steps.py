"""Rows in 8 bits, bit by bit: scale = max |y| / 127 and q = y / scale rounded to nearest, ties to even, each one fp32 operation on y in fp32, which
is h * rstd * gamma in this order.  The rows are made of values next to the border between two steps, where another order of the operations, or
another division, gives another step."""
import numpy as np
import pytest

import fastconv_amd as F
import state_space as S
import tokens as K

pytestmark = pytest.mark.gpu

f32 = np.float32


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


def steps(y):
    """scale and q of fp32 rows, in fp32, and how far y / scale lies from the nearest border."""
    scale = np.abs(y).max(axis=1) / f32(127)
    exact = y / scale[:, None]
    assert y.dtype == scale.dtype == exact.dtype == f32
    return scale, np.rint(exact), np.abs(exact - np.floor(exact) - f32(0.5))


def border_rows(rng, rows, C, dtype):
    """h and gamma, whose products of a row lie half a step from a whole one, within the rounding of h (fp32) or of gamma (16 bits: rows are powers of
    two times the first, each of which has another rstd)."""
    k = (rng.integers(-126, 126, C) + 0.5) / 127
    k[C // 3] = 1.0
    if dtype == "f32":
        gamma = (1 + 0.2 * rng.standard_normal(C)).astype(f32)
        return K.to_type((k / gamma) * rng.uniform(0.5, 8, (rows, 1)), dtype)[1], gamma
    h = K.to_type(rng.uniform(0.5, 2, C) * rng.choice((-1, 1), C), dtype)[1]
    return h * 2.0 ** rng.integers(-8, 9, (rows, 1)), (k / h).astype(f32)


# every number of wavefronts of a row and of accesses that are kept, and rows that are read again
@pytest.mark.parametrize("rows,C,dtype", [(5, 7, "f32"), (40, 200, "f32"), (300, 500, "bf16"), (9, 1000, "f32"), (64, 2046, "f16"), (200, 2048, "bf16"),
                                          (33, 4096, "f32"), (12, 8192, "bf16"), (6, 9001, "f32"), (3, 40001, "f32"), (2, 40008, "bf16")])
def test_values_on_the_border_between_two_steps(lib, rows, C, dtype):
    rng = np.random.default_rng(rows + C)
    mark = lib.mark()
    try:
        print("steps of rows", rows, C, dtype, flush=True)
        h, gamma = border_rows(rng, rows, C, dtype)
        x, g = K.Dev(lib, (rows, C), dtype, None, h), K.floats(lib, gamma)
        assert np.array_equal(x.values, h)
        plan = lib.rms_norm_plan(F.RmsNormShape.packed(rows, C, K.TYPES[dtype], 1e-5))
        y, rstd, scale, q = K.Dev(lib, (rows, C), dtype), K.Dev(lib, (rows,), "f32"), K.Dev(lib, (rows,), "f32"), lib.alloc(rows * C)
        lib.rms_norm(plan, x.ptr, g, y.ptr, rstd=rstd.ptr)
        lib.rms_norm_int8(plan, x.ptr, g, q, scale.ptr)
        values = (h.astype(f32) * rstd.get().astype(f32)[:, None]) * gamma
        if dtype == "f32":
            assert np.array_equal(y.get(), values)
        want_scale, want, border = steps(values)
        # k + 0.5 is off by a few last places of up to 127: 127 * 8 * 2^-24
        assert (border < 6.1e-5).mean() > 0.9 - 1 / C
        got = lib.download(q, (rows, C), np.int8)
        assert np.array_equal(scale.get(), want_scale)
        assert np.array_equal(got, want), "%d of %d steps" % ((got != want).sum(), got.size)
        # the same rows by themselves
        dy = K.Dev(lib, (rows, C), "f32", None, values)
        lib.quantize_rows(rows, C, F.F32, dy.ptr, q, scale.ptr)
        assert np.array_equal(scale.get(), want_scale) and np.array_equal(lib.download(q, (rows, C), np.int8), want)
    finally:
        lib.release(mark)


@pytest.mark.parametrize("C", [40, 2048, 9001, 40001])
@pytest.mark.parametrize("size,eps", [(2.0 ** -122, 1e-8), (1e-36, 1e-8), (2e-38, 1e-12), (1e-40, 1e-19), (3e-32, 1e-5), (2e-36, 3e-7)])
def test_small_rows_beside_a_small_eps(lib, C, size, eps):
    """Rows far below the root of eps, whose results are still numbers: the norm multiplies them by up to 1 / sqrt(eps), and 127 over their own largest
    value would be infinite.  y errs by its two products and rstd's rounding, which its scale shares: 8 last places of up to 127 as elsewhere, and
    subnormal values of x are exact."""
    rng = np.random.default_rng(C)
    mark = lib.mark()
    try:
        print("small rows", C, size, eps, flush=True)
        h = K.to_type(size * rng.uniform(0.5, 2, (3, C)) * rng.choice((-1, 1), (3, C)), "f32")[1]
        gamma = (1 + 0.2 * rng.standard_normal(C)).astype(f32)
        x, scale, q = K.Dev(lib, (3, C), "f32", None, h), K.Dev(lib, (3,), "f32"), lib.alloc(3 * C)
        lib.rms_norm_int8(lib.rms_norm_plan(F.RmsNormShape.packed(3, C, F.F32, eps)), x.ptr, K.floats(lib, gamma), q, scale.ptr)
        want, _ = S.rms_norm(h, gamma.astype(np.float64), np.float64(f32(eps)))
        top = np.abs(want).max(axis=1)
        assert (top > 2.0 ** -109).all()      # rows that the interface promises to round
        S.close(scale.get(), top / 127, 56 * K.EPS * top / 127, "scale")
        S.close(lib.download(q, (3, C), np.int8).astype(np.float64), want * (127 / top)[:, None], 0.5 + 127 * 8 * K.EPS, "q")
    finally:
        lib.release(mark)
