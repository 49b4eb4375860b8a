"""RMS norm with a residual, in the rows' type and in 8 bits, against the formulas in 64 bits.

The sum is rounded to its type from the fp32 sum, as here: equal bits.  The sum of squares errs by fewer than 80 last places (32 values of a thread in
order, six and sixteen joins; streamed rows 16 more), its root by half of that, and each product by one: 48 last places of rstd, 56 of y.  In 8 bits
a value is off by half a step and by 127 * 8 last places of the row's largest, its scale by 56 last places.  Gradients: the mean along xhat is a sum of C terms."""
import numpy as np
import pytest

import fastconv_amd as F
import state_space as S
import tokens as K

pytestmark = pytest.mark.gpu

NORM, VALUE = 48 * K.EPS, 56 * K.EPS
E = 1e-5


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


def rows_of(rng, rows, C):
    return rng.standard_normal((rows, C)) * np.exp(0.7 * rng.standard_normal(C))


def make(L, rng, rows, C, dtype, residual=True, gap=0, offset=0, values=None, eps=E):
    x = rows_of(rng, rows, C) if values is None else values
    pitch = C + gap
    dx = K.Dev(L, (rows, C), dtype, (pitch, 1), x, offset)
    dr = K.Dev(L, (rows, C), dtype, (pitch, 1), 2 * rows_of(rng, rows, C), offset) if residual else None
    shape = F.RmsNormShape(rows, C, K.TYPES[dtype], eps, pitch, pitch, C if residual else pitch, C)
    h = dx.values if dr is None else K.to_type((dx.values + dr.values).astype(np.float32), dtype)[1]
    gamma = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32)
    return dx, dr, L.rms_norm_plan(shape), h, gamma


CASES = [  # rows, C, dtype, residual, gap, offset
    (1, 1, "f32", True, 0, 0),
    (1, 8, "bf16", False, 0, 0),
    (3, 7, "f16", True, 0, 0),
    (5, 96, "bf16", True, 8, 0),
    (1, 2048, "bf16", True, 0, 0),
    (7, 2046, "f16", True, 0, 0),          # two values an access
    (4, 771, "f32", True, 5, 0),
    (2, 771, "bf16", False, 3, 1),         # rows that begin on odd elements
    (3, 4096, "f32", True, 0, 0),
    (2, 8192, "bf16", True, 0, 0),
    (2, 8200, "bf16", True, 8, 0),         # sixteen wavefronts
    (2, 4097, "f32", True, 0, 0),
    (2, 33000, "bf16", True, 0, 0),        # read twice
    (3, 5003, "f16", True, 0, 0),
    (2, 40001, "f32", False, 0, 0),
    (1500, 64, "bf16", True, 0, 0),
    (1027, 2048, "f16", True, 0, 0),
    (9001, 24, "f32", True, 0, 0),
    (2500, 4104, "bf16", True, 0, 0),      # more rows than workgroups
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(lib, case):
    rows, C, dtype, residual, gap, offset = case
    rng = np.random.default_rng(rows + C)
    mark = lib.mark()
    try:
        print("rms norm", case, flush=True)
        dx, dr, plan, h, gamma = make(lib, rng, rows, C, dtype, residual, gap, offset)
        y, total = K.Dev(lib, (rows, C), dtype, None, None, offset), K.Dev(lib, (rows, C), dtype, None, None, offset) if residual else None
        r, g = K.Dev(lib, (rows,), "f32"), K.floats(lib, gamma)
        lib.rms_norm(plan, dx.ptr, g, y.ptr, dr.ptr if residual else None, total.ptr if residual else None, r.ptr)
        want, rstd = S.rms_norm(h, gamma.astype(np.float64), E)
        if residual:
            assert np.array_equal(total.get(), h)
        S.close(r.get(), rstd[:, 0], NORM * rstd[:, 0], "rstd")
        S.close(y.get(), want, (K.ROUND[dtype] + VALUE) * np.abs(want) + K.TINY[dtype], "y")
        # 8 bits
        q, scale = lib.upload_raw(np.full((rows, C), 0x5a, np.int8)), K.Dev(lib, (rows,), "f32")
        again = K.Dev(lib, (rows, C), dtype, None, None, offset) if residual else None
        lib.rms_norm_int8(plan, dx.ptr, g, q, scale.ptr, dr.ptr if residual else None, again.ptr if residual else None)
        if residual:
            assert np.array_equal(again.get(), h)
        top = np.abs(want).max(axis=1)
        S.close(scale.get(), top / 127, VALUE * top / 127, "scale")
        S.close(lib.download(q, (rows, C), np.int8).astype(np.float64), want * (127 / top)[:, None], 0.5 + 127 * 8 * K.EPS, "q")
        # backward
        dy = K.Dev(lib, (rows, C), dtype, None, rng.standard_normal((rows, C)), offset)
        ds = K.Dev(lib, (rows, C), dtype, None, rng.standard_normal((rows, C)), offset) if residual else None
        out, dgamma = K.Dev(lib, (rows, C), dtype, dx.strides, None, offset), K.Dev(lib, (C,), "f32")
        src = total.ptr if residual else dx.ptr
        ws = lib.alloc(plan.ws_backward_bytes)
        lib.rms_norm_backward(plan, dy.ptr, src, g, r.ptr, out.ptr, dgamma.ptr, ds.ptr if residual else None, ws)
        want, wg = S.rms_norm_backward(dy.values, h, gamma.astype(np.float64), rstd, ds.values if residual else None)
        gd, xhat = np.abs(dy.values * gamma), np.abs(h * rstd)
        along = (gd * xhat).mean(axis=1, keepdims=True)
        tol = rstd * ((NORM + 6 * K.EPS) * gd + xhat * along * (3 * NORM + K.EPS * (16 + 2 * np.sqrt(C)))) + 2 * K.EPS * np.abs(want)
        S.close(out.get(), want, K.ROUND[dtype] * np.abs(want) + tol + K.TINY[dtype], "dx")
        S.close(dgamma.get(), wg, (NORM + K.EPS * (8 + 2 * np.sqrt(rows))) * np.abs(dy.values * xhat).sum(axis=0) + 1e-30, "dgamma")
        # again: the same bits; without dgamma no workspace
        other = K.Dev(lib, (rows, C), dtype, dx.strides, None, offset)
        lib.rms_norm_backward(plan, dy.ptr, src, g, r.ptr, other.ptr, None, ds.ptr if residual else None, None)
        assert np.array_equal(other.get(), out.get())
    finally:
        lib.release(mark)


def test_in_place(lib):
    """The sum over the residual, the result over x; a row that is read twice among them."""
    rng = np.random.default_rng(1)
    for C in (64, 2048, 40001):
        mark = lib.mark()
        dx, dr, plan, h, gamma = make(lib, rng, 3, C, "f32")
        shape = F.RmsNormShape.packed(3, C, F.F32, E)
        plan = lib.rms_norm_plan(shape)
        print("rms norm in place", C, flush=True)
        lib.rms_norm(plan, dx.ptr, None, dx.ptr, dr.ptr, dr.ptr)
        want, _ = S.rms_norm(h, 1.0, E)
        assert np.array_equal(dr.get(), h)
        S.close(dx.get(), want, (K.ROUND["f32"] + VALUE) * np.abs(want), "y")
        # the gradient over that of the sum
        rstd, ds = K.floats(lib, 1 / np.sqrt((h ** 2).mean(axis=1) + E)), K.Dev(lib, (3, C), "f32", None, rng.standard_normal((3, C)))
        before, dy = ds.values.copy(), K.Dev(lib, (3, C), "f32", None, rng.standard_normal((3, C)))
        out = K.Dev(lib, (3, C), "f32")
        lib.rms_norm_backward(plan, dy.ptr, dr.ptr, None, rstd, out.ptr, None, ds.ptr)
        lib.rms_norm_backward(plan, dy.ptr, dr.ptr, None, rstd, ds.ptr, None, ds.ptr)
        assert np.array_equal(out.get(), ds.get()) and not np.array_equal(ds.get(), before)
        lib.release(mark)


@pytest.mark.parametrize("C", [40, 2048, 40001])
def test_largest_and_smallest_values(lib, C):
    """Squares that overflow fp32, or vanish where there is no eps; rows of zeros."""
    rng = np.random.default_rng(C)
    for size, eps in ((1e30, 1e-5), (3e37, 0.0), (1e-30, 0.0), (1e-36, 1e-30), (1e-3, 0.0)):
        mark = lib.mark()
        values = size * rng.uniform(0.5, 2, (2, C)) * rng.choice((-1, 1), (2, C))
        dx, _, plan, h, gamma = make(lib, rng, 2, C, "f32", False, values=values, eps=eps)
        y, q, scale = K.Dev(lib, (2, C), "f32"), lib.alloc(2 * C), K.Dev(lib, (2,), "f32")
        print("rms norm", C, size, eps, flush=True)
        lib.rms_norm(plan, dx.ptr, K.floats(lib, gamma), y.ptr)
        want, _ = S.rms_norm(h, gamma.astype(np.float64), np.float64(np.float32(eps)))
        S.close(y.get(), want, (K.ROUND["f32"] + VALUE) * np.abs(want), "y of %g" % size)
        lib.rms_norm_int8(plan, dx.ptr, K.floats(lib, gamma), q, scale.ptr)
        top = np.abs(want).max(axis=1)
        S.close(scale.get(), top / 127, VALUE * top / 127, "scale of %g" % size)
        S.close(lib.download(q, (2, C), np.int8).astype(np.float64), want * (127 / top)[:, None], 0.5 + 127 * 8 * K.EPS, "q of %g" % size)
        lib.release(mark)


def test_rows_of_zeros_and_rows_that_are_not_finite(lib):
    """A row keeps what it has to itself."""
    for C in (33, 2048, 40001):
        for dtype in ("f32", "bf16"):
            mark = lib.mark()
            x = np.random.default_rng(0).standard_normal((5, C))
            x[1] = 0
            x[2, C // 2] = np.nan
            x[3, C - 1] = -np.inf
            dx = K.Dev(lib, (5, C), dtype, None, x)
            plan = lib.rms_norm_plan(F.RmsNormShape.packed(5, C, K.TYPES[dtype], E))
            y, q, scale = K.Dev(lib, (5, C), dtype), lib.alloc(5 * C), K.Dev(lib, (5,), "f32")
            print("rms norm, not finite", C, dtype, flush=True)
            lib.rms_norm(plan, dx.ptr, None, y.ptr)
            got = y.get()
            want, _ = S.rms_norm(dx.values, 1.0, E)
            for i in (0, 4):
                S.close(got[i], want[i], (K.ROUND[dtype] + VALUE) * np.abs(want[i]) + K.TINY[dtype], "y")
            assert not got[1].any() and np.isnan(got[2]).all() and np.isnan(got[3, C - 1])
            for call in (lambda: lib.rms_norm_int8(plan, dx.ptr, None, q, scale.ptr),
                         lambda: lib.quantize_rows(5, C, K.TYPES[dtype], dx.ptr, q, scale.ptr)):
                call()
                s, b = scale.get(), lib.download(q, (5, C), np.int8)
                assert s[1] == 0 and np.isnan(s[2]) and np.isnan(s[3]) and not b[1:4].any()
                assert np.abs(b[0]).max() == 127 and np.abs(b[4]).max() == 127
            lib.release(mark)


@pytest.mark.parametrize("rows,C,dtype,gap,q_gap", [(1, 5, "f32", 0, 0), (3, 1000, "bf16", 0, 8), (4, 771, "f16", 2, 5), (1025, 2048, "bf16", 0, 0),
                                                    (2, 20001, "f32", 0, 0), (40, 256, "bf16", 8, 3)])
def test_quantized_rows(lib, rows, C, dtype, gap, q_gap):
    rng = np.random.default_rng(C)
    mark = lib.mark()
    x = K.Dev(lib, (rows, C), dtype, (C + gap, 1), rows_of(rng, rows, C))
    pitch = C + q_gap
    before = np.full(rows * pitch + 64, 0x5a, np.int8)
    q, scale = lib.upload_raw(before), K.Dev(lib, (rows,), "f32")
    print("quantize rows", rows, C, dtype, flush=True)
    lib.quantize_rows(rows, C, K.TYPES[dtype], x.ptr, q, scale.ptr, C + gap, pitch)
    got = lib.download(q, before.shape, np.int8)
    top = np.abs(x.values).max(axis=1)
    S.close(scale.get(), top / 127, 2 * K.EPS * top, "scale")
    held = got[:rows * pitch].reshape(rows, pitch)
    S.close(held[:, :C].astype(np.float64), x.values * (127 / top)[:, None], 0.5 + 127 * 3 * K.EPS, "q")
    assert (held[:, C:] == 0x5a).all() and (got[rows * pitch:] == 0x5a).all()
    # ties go to even: a row whose scale is exactly one
    row = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 3.25]])
    t = K.Dev(lib, (1, 8), "f32", None, row)
    lib.quantize_rows(1, 8, F.F32, t.ptr, q, scale.ptr)
    assert list(lib.download(q, (8,), np.int8)) == [127, 0, 2, 2, 0, -2, -126, 3]
    lib.release(mark)


def test_gradient_against_differences(lib):
    rows, C = 6, 48
    rng = np.random.default_rng(5)
    dx, dr, plan, h, gamma = make(lib, rng, rows, C, "f32")
    total, y, rstd = (K.Dev(lib, s, "f32") for s in ((rows, C), (rows, C), (rows,)))
    g = K.floats(lib, gamma)
    lib.rms_norm(plan, dx.ptr, g, y.ptr, dr.ptr, total.ptr, rstd.ptr)
    w, ws = (K.Dev(lib, (rows, C), "f32", None, rng.standard_normal((rows, C))) for _ in range(2))
    out, dgamma = K.Dev(lib, (rows, C), "f32"), K.Dev(lib, (C,), "f32")
    lib.rms_norm_backward(plan, w.ptr, total.ptr, g, rstd.ptr, out.ptr, dgamma.ptr, ws.ptr, lib.alloc(plan.ws_backward_bytes))
    loss = lambda a, c: (S.rms_norm(a, c, E)[0] * w.values).sum() + (a * ws.values).sum()  # noqa: E731
    u, ug, e = rng.standard_normal((rows, C)), rng.standard_normal(C), 1e-4
    gamma = gamma.astype(np.float64)
    diff = (loss(h + e * u, gamma + e * ug) - loss(h - e * u, gamma - e * ug)) / (2 * e)
    along = (out.get() * u).sum() + (dgamma.get() * ug).sum()
    # fp32 sums of a few hundred terms of order one, and e^2 times a third derivative of that order
    assert abs(diff - along) <= 1e-4 * (np.abs(out.get() * u).sum() + np.abs(dgamma.get() * ug).sum())


def test_in_a_graph(lib):
    """Recorded, replayed on new values between eager calls: the same bits as the eager calls."""
    rng = np.random.default_rng(9)
    rows, C = 40, 1024
    plan = lib.rms_norm_plan(F.RmsNormShape.packed(rows, C, F.F32, E))
    x, r = lib.alloc(4 * rows * C), lib.alloc(4 * rows * C)
    q, s, total, q2, s2, total2 = (lib.alloc(n) for n in 2 * (rows * C, 4 * rows, 4 * rows * C))
    lib.graph_begin()
    lib.rms_norm_int8(plan, x, None, q, s, r, total)
    g = lib.graph_end()
    for turn in range(3):
        lib.upload_into(x, rows_of(rng, rows, C))
        lib.upload_into(r, rows_of(rng, rows, C))
        print("rms norm in a graph, replay", turn, flush=True)
        lib.rms_norm_int8(plan, x, None, q2, s2, r, total2)
        lib.graph_launch(g)
        lib.sync()
        assert np.array_equal(lib.download(q, (rows, C), np.int8), lib.download(q2, (rows, C), np.int8))
        assert np.array_equal(lib.download(s, (rows,)), lib.download(s2, (rows,)))
        assert np.array_equal(lib.download(total, (rows, C)), lib.download(total2, (rows, C)))
    lib.graph_destroy(g)


def test_refusals(lib):
    rows, C = 4, 16
    p = [lib.alloc(4096) for _ in range(6)]
    plan = lib.rms_norm_plan(F.RmsNormShape.packed(rows, C, F.BF16))
    odd = p[0].value + 1
    bad = lib.rms_norm_plan(F.RmsNormShape(rows, C, F.BF16, 1e-5, C, C, C, C - 1))
    no_sum = lib.rms_norm_plan(F.RmsNormShape(rows, C, F.BF16, 1e-5, C, C, C - 1, C))
    shared = lib.rms_norm_plan(F.RmsNormShape(rows, C, F.BF16, 1e-5, 0, C, C, C))
    other = F.RmsNormPlan.from_buffer_copy(plan)
    other.parts += 1
    calls = [
        lambda: lib.rms_norm(plan, None, None, p[1]), lambda: lib.rms_norm(plan, p[0], None, None), lambda: lib.rms_norm(plan, odd, None, p[1]),
        lambda: lib.rms_norm(plan, p[0], p[1].value + 2, p[2]), lambda: lib.rms_norm(bad, p[0], None, p[1]),
        lambda: lib.rms_norm(no_sum, p[0], None, p[1], p[2], p[3]), lambda: lib.rms_norm(other, p[0], None, p[1]),
        lambda: lib.rms_norm_int8(plan, p[0], None, None, p[2]), lambda: lib.rms_norm_int8(plan, p[0], None, p[1], None),
        lambda: lib.rms_norm_int8(plan, p[0], None, p[1], p[2].value + 1), lambda: lib.rms_norm_int8(bad, p[0], None, p[1], p[2]),
        lambda: lib.rms_norm_backward(plan, p[0], p[1], None, None, p[3]), lambda: lib.rms_norm_backward(plan, p[0], p[1], None, p[2], p[3], p[4]),
        lambda: lib.rms_norm_backward(shared, p[0], p[1], None, p[2], p[3]),
        lambda: lib.quantize_rows(0, C, F.F32, p[0], p[1], p[2]), lambda: lib.quantize_rows(rows, C, 3, p[0], p[1], p[2]),
        lambda: lib.quantize_rows(rows, C, F.F32, p[0], p[1], p[2], q_row=C - 1), lambda: lib.quantize_rows(rows, C, F.F32, odd, p[1], p[2]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(F.FastConvError) as e:
            call()
        assert e.value.status == -1, i
    with pytest.raises(F.FastConvError) as e:
        lib.quantize_rows(1, (1 << 20) + 1, F.F32, p[0], p[1], p[2])
    assert e.value.status == -6


@pytest.mark.parametrize("case", [  # widths on both sides of where another number of accesses is kept, more rows than there are workgroups for
    (17000, 72, "bf16", True, 0, 0), (4500, 256, "f32", True, 0, 0), (4500, 257, "f32", True, 3, 1), (9000, 512, "f16", True, 0, 0), (9000, 513, "bf16", True, 0, 0),
    (2100, 1024, "bf16", False, 0, 0), (2100, 1025, "bf16", True, 0, 0), (2100, 516, "f32", True, 0, 0)], ids=lambda c: "-".join(map(str, c)))
def test_widths_of_each_form(lib, case):
    test_forward_and_backward(lib, case)
