"""Short causal convolutions of single channels, forward and backward, against the formulas in 64 bits (bounds: state_space.causal_conv)."""
import numpy as np
import pytest

import fastconv_amd as F
import state_space as S
import tokens as K

pytestmark = pytest.mark.gpu

ACTS = {"none": F.ACT_NONE, "silu": F.ACT_SILU}


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


CASES = [  # B, T, C, taps, dtype, act, bias, carry, lengths, gap
    (1, 1, 1, 2, "f32", "none", True, True, None, 0),
    (64, 1, 256, 4, "bf16", "silu", True, True, None, 0),
    (3, 1, 40, 4, "f16", "silu", True, True, [1, 0, 1], 0),
    (2, 2, 24, 4, "bf16", "silu", True, True, None, 0),           # fewer tokens than taps
    (2, 3, 10, 8, "f32", "silu", True, True, [3, 1], 0),
    (1, 100, 64, 4, "bf16", "silu", True, False, None, 0),
    (2, 77, 63, 3, "f16", "silu", False, True, None, 0),          # odd channels
    (2, 130, 96, 4, "bf16", "none", True, True, [130, 57], 32),   # rows with a gap
    (3, 130, 96, 5, "f32", "silu", True, True, [0, 2, 4], 3),
    (2, 65, 48, 7, "bf16", "silu", True, True, None, 0),
    (2, 50, 34, 6, "f16", "none", False, True, [50, 31], 0),
    (4, 33, 1002, 2, "bf16", "silu", True, True, None, 0),        # two values an access
    (1, 5000, 16, 4, "f32", "silu", True, True, None, 0),         # cut into walks
    (5, 1225, 8, 8, "bf16", "silu", True, True, [1225, 1224, 0, 1, 700], 0),
    (2, 3136, 512, 4, "bf16", "silu", True, False, None, 0),
    (1, 40, 5, 2, "f16", "silu", True, True, [-3], 0),
    (1, 40, 5, 3, "f16", "silu", True, True, [99], 0),
]


def strided(shape, gap):
    B, T, C = shape
    return (T * (C + gap) + 5 * (gap > 0), C + gap, 1)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(lib, case):
    B, T, C, taps, dtype, act, bias, carry, lengths, gap = case
    rng = np.random.default_rng(B + T + C + taps)
    mark = lib.mark()
    try:
        print("causal conv", case, flush=True)
        n = S.lengths_of(lengths, B, T)
        values = rng.standard_normal((B, T, C))
        for b in range(B):
            values[b, n[b]:] = np.nan      # not read
        x = K.Dev(lib, (B, T, C), dtype, strided((B, T, C), gap), values)
        clean = np.nan_to_num(x.values)
        w, b0 = (rng.standard_normal((C, taps)) / np.sqrt(taps)).astype(np.float32), (0.3 * rng.standard_normal(C)).astype(np.float32) if bias else None
        dw_, db_ = K.floats(lib, w), K.floats(lib, b0) if bias else None
        w, b0 = w.astype(np.float64), b0.astype(np.float64) if bias else None
        state = K.Dev(lib, (B, taps - 1, C), dtype, None, rng.standard_normal((B, taps - 1, C))) if carry else None
        y, after = K.Dev(lib, (B, T, C), dtype), K.Dev(lib, (B, taps - 1, C), dtype)
        shape = F.CausalConvShape(B, T, C, taps, K.TYPES[dtype], ACTS[act], x.strides[0], x.strides[1], T * C, C)
        plan = lib.causal_conv_plan(shape)
        dl = lib.upload_raw(np.array(lengths, np.int32)) if lengths else None
        lib.causal_conv(plan, x.ptr, dw_, db_, y.ptr, state.ptr if carry else None, after.ptr, dl)
        first = state.values if carry else None
        want, last, z, tz = S.causal_conv(clean, w, b0, act == "silu", first, lengths)
        tol = 1.1 * tz + (8 + 2 * np.abs(z)) * K.EPS * np.abs(want) if act == "silu" else tz
        S.close(y.get(), want, K.ROUND[dtype] * np.abs(want) + tol + K.TINY[dtype], "y")
        assert np.array_equal(after.get(), last)
        if carry:      # the state over the one before
            again = K.Dev(lib, (B, T, C), dtype)
            lib.causal_conv(plan, x.ptr, dw_, db_, again.ptr, state.ptr, state.ptr, dl)
            assert np.array_equal(state.get(), last) and np.array_equal(again.get(), y.get())
            state = K.Dev(lib, (B, taps - 1, C), dtype, None, first)
        grads = rng.standard_normal((B, T, C))
        for b in range(B):
            grads[b, n[b]:] = np.nan
        dy = K.Dev(lib, (B, T, C), dtype, None, grads)
        up = np.nan_to_num(dy.values)
        dlast = K.Dev(lib, (B, taps - 1, C), dtype, None, rng.standard_normal((B, taps - 1, C))) if carry else None
        dx, dfirst = K.Dev(lib, (B, T, C), dtype, x.strides), K.Dev(lib, (B, taps - 1, C), dtype)
        dw, db = K.Dev(lib, (C, taps), "f32"), K.Dev(lib, (C,), "f32")
        space = lib.alloc(plan.ws_backward_bytes)
        lib.causal_conv_backward(plan, dy.ptr, x.ptr, dw_, db_, dx.ptr, dw.ptr, db.ptr, state.ptr if carry else None,
                                 dlast.ptr if carry else None, dfirst.ptr, dl, space)
        got, tol = S.causal_conv_backward(up, clean, w, b0, act == "silu", first, dlast.values if carry else None, lengths)
        for name, dev, a, t, kind in zip(("dx", "dw", "dbias", "dstate"), (dx, dw, db, dfirst), got, tol, (dtype, "f32", "f32", dtype)):
            S.close(dev.get(), a, K.ROUND[kind] * np.abs(a) + t + K.TINY[kind], name)
        # again, each part alone: the same bits
        dx2, dw2, db2 = K.Dev(lib, (B, T, C), dtype, x.strides), K.Dev(lib, (C, taps), "f32"), K.Dev(lib, (C,), "f32")
        args = (state.ptr if carry else None, dlast.ptr if carry else None, None, dl)
        lib.causal_conv_backward(plan, dy.ptr, x.ptr, dw_, db_, dx2.ptr, None, None, *args)
        assert np.array_equal(dx2.get(), dx.get())
        lib.causal_conv_backward(plan, dy.ptr, x.ptr, dw_, db_, dx2.ptr, dw2.ptr, None, *args, space)
        lib.causal_conv_backward(plan, dy.ptr, x.ptr, dw_, db_, dx2.ptr, None, db2.ptr, *args, space)
        assert np.array_equal(dw2.get(), dw.get()) and np.array_equal(db2.get(), db.get())
    finally:
        lib.release(mark)


def test_tokens_one_by_one_are_the_prompt(lib):
    """The same sums in the same order: the same bits, whatever the sequence is cut into."""
    rng = np.random.default_rng(1)
    B, T, C = 2, 23, 72
    for taps in (2, 3, 4, 6):
        for dtype in ("f32", "bf16"):
            x = K.Dev(lib, (B, T, C), dtype, None, rng.standard_normal((B, T, C)))
            w, bias = K.floats(lib, rng.standard_normal((C, taps))), K.floats(lib, rng.standard_normal(C))
            whole, parts = K.Dev(lib, (B, T, C), dtype), K.Dev(lib, (B, T, C), dtype)
            state, one = K.Dev(lib, (B, taps - 1, C), dtype), K.Dev(lib, (B, taps - 1, C), dtype)
            es = 4 if dtype == "f32" else 2
            lib.causal_conv(lib.causal_conv_plan(F.CausalConvShape.packed(B, T, C, taps, K.TYPES[dtype])), x.ptr, w, bias, whole.ptr, None, state.ptr)
            at = 0
            print("causal conv, token by token", taps, dtype, flush=True)
            for n in (1, 9, 2, 1, 1, 9):
                plan = lib.causal_conv_plan(F.CausalConvShape(B, n, C, taps, K.TYPES[dtype], F.ACT_SILU, T * C, C, T * C, C))
                lib.causal_conv(plan, x.ptr + at * C * es, w, bias, parts.ptr + at * C * es, one.ptr if at else None, one.ptr)
                at += n
            assert at == T and np.array_equal(whole.get(), parts.get()) and np.array_equal(state.get(), one.get())


def test_what_is_not_finite_stays_in_its_window(lib):
    B, T, C, taps = 1, 60, 16, 5
    values = np.random.default_rng(2).standard_normal((B, T, C))
    values[0, 20, 3], values[0, 30, 4] = np.nan, np.inf
    x = K.Dev(lib, (B, T, C), "f32", None, values)
    w = np.ones((C, taps), np.float32)
    y = K.Dev(lib, (B, T, C), "f32")
    lib.causal_conv(lib.causal_conv_plan(F.CausalConvShape.packed(B, T, C, taps, F.F32, F.ACT_NONE)), x.ptr, K.floats(lib, w), None, y.ptr)
    bad = ~np.isfinite(y.get())
    want = np.zeros(bad.shape, bool)
    want[0, 20:25, 3] = want[0, 30:35, 4] = True
    assert np.array_equal(bad, want)


def test_shared_input(lib):
    """One sequence for all (stride 0) is an input, and is no gradient."""
    rng = np.random.default_rng(3)
    T, C, taps = 20, 24, 4
    x, w = K.Dev(lib, (1, T, C), "f32", None, rng.standard_normal((1, T, C))), K.floats(lib, rng.standard_normal((C, taps)))
    y, one = K.Dev(lib, (3, T, C), "f32"), K.Dev(lib, (1, T, C), "f32")
    plan = lib.causal_conv_plan(F.CausalConvShape(3, T, C, taps, F.F32, F.ACT_SILU, 0, C, T * C, C))
    lib.causal_conv(plan, x.ptr, w, None, y.ptr)
    lib.causal_conv(lib.causal_conv_plan(F.CausalConvShape.packed(1, T, C, taps)), x.ptr, w, None, one.ptr)
    assert np.array_equal(y.get(), np.repeat(one.get(), 3, axis=0))
    with pytest.raises(F.FastConvError) as e:
        lib.causal_conv_backward(plan, y.ptr, x.ptr, w, None, one.ptr)
    assert e.value.status == -1


def test_gradient_against_differences(lib):
    rng = np.random.default_rng(5)
    B, T, C, taps, e = 2, 19, 12, 4, 1e-4
    draw = lambda *s: K.Dev(lib, s, "f32", None, rng.standard_normal(s))  # noqa: E731
    x, state, dy, dlast = draw(B, T, C), draw(B, taps - 1, C), draw(B, T, C), draw(B, taps - 1, C)
    w, bias = rng.standard_normal((C, taps)).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    out = [K.Dev(lib, s, "f32") for s in ((B, T, C), (C, taps), (C,), (B, taps - 1, C))]
    plan = lib.causal_conv_plan(F.CausalConvShape.packed(B, T, C, taps))
    lib.causal_conv_backward(plan, dy.ptr, x.ptr, K.floats(lib, w), K.floats(lib, bias), out[0].ptr, out[1].ptr, out[2].ptr, state.ptr, dlast.ptr,
                             out[3].ptr, None, lib.alloc(plan.ws_backward_bytes))

    def loss(a, b, c, d):
        y, after, _, _ = S.causal_conv(a, b, c, True, d)
        return (y * dy.values).sum() + (after * dlast.values).sum()
    at = [x.values, w.astype(np.float64), bias.astype(np.float64), state.values]
    u = [rng.standard_normal(a.shape) for a in at]
    diff = (loss(*(a + e * d for a, d in zip(at, u))) - loss(*(a - e * d for a, d in zip(at, u)))) / (2 * e)
    along = [(o.get() * d) for o, d in zip(out, u)]
    assert abs(diff - sum(a.sum() for a in along)) <= 1e-4 * np.sqrt(sum((a ** 2).sum() for a in along)) * 10


def test_in_a_graph(lib):
    rng = np.random.default_rng(7)
    B, T, C, taps = 2, 300, 64, 4
    plan = lib.causal_conv_plan(F.CausalConvShape.packed(B, T, C, taps))
    x, dy = lib.alloc(4 * B * T * C), lib.alloc(4 * B * T * C)
    w = K.floats(lib, rng.standard_normal((C, taps)))
    sets = [[lib.alloc(4 * n) for n in (B * T * C, B * T * C, C * taps, C)] + [lib.alloc(plan.ws_backward_bytes)] for _ in range(2)]

    def both(s):
        lib.causal_conv(plan, x, w, None, s[0])
        lib.causal_conv_backward(plan, dy, x, w, None, s[1], s[2], s[3], ws=s[4])
    lib.graph_begin()
    both(sets[0])
    g = lib.graph_end()
    for turn in range(3):
        lib.upload_into(x, rng.standard_normal((B, T, C)))
        lib.upload_into(dy, rng.standard_normal((B, T, C)))
        print("causal conv in a graph, replay", turn, flush=True)
        both(sets[1])
        lib.graph_launch(g)
        lib.sync()
        for i, n in enumerate((B * T * C, B * T * C, C * taps, C)):
            assert np.array_equal(lib.download(sets[0][i], (n,)), lib.download(sets[1][i], (n,)))
    lib.graph_destroy(g)


def test_refusals(lib):
    p = [lib.alloc(1 << 16) for _ in range(6)]
    plan = lib.causal_conv_plan(F.CausalConvShape.packed(2, 8, 16, 4, F.BF16))
    other = F.CausalConvPlan.from_buffer_copy(plan)
    other.walks += 1
    over = lib.causal_conv_plan(F.CausalConvShape(2, 8, 16, 4, F.BF16, F.ACT_SILU, 128, 16, 128, 15))
    calls = [lambda: lib.causal_conv(plan, None, p[1], None, p[2]), lambda: lib.causal_conv(plan, p[0], None, None, p[2]),
             lambda: lib.causal_conv(plan, p[0], p[1], None, None), lambda: lib.causal_conv(plan, p[0].value + 1, p[1], None, p[2]),
             lambda: lib.causal_conv(plan, p[0], p[1].value + 2, None, p[2]), lambda: lib.causal_conv(plan, p[0], p[1], None, p[2], p[3].value + 1),
             lambda: lib.causal_conv(plan, p[0], p[1], None, p[2], lengths=p[3].value + 2), lambda: lib.causal_conv(other, p[0], p[1], None, p[2]),
             lambda: lib.causal_conv(over, p[0], p[1], None, p[2]), lambda: lib.causal_conv_backward(plan, p[0], p[1], p[2], None, None),
             lambda: lib.causal_conv_backward(plan, p[0], p[1], p[2], None, p[3], p[4])]
    for i, call in enumerate(calls):
        with pytest.raises(F.FastConvError) as e:
            call()
        assert e.value.status == -1, i


@pytest.mark.parametrize("taps", [5, 6, 7, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_taps_over_long_walks(lib, taps, dtype):
    """A walk of many steps whose window reaches further back than the rows that are read at once, and the state over the one before."""
    B, T, C = 64, 45, 2 * 4096 + 1
    rng = np.random.default_rng(taps)
    mark = lib.mark()
    try:
        print("causal conv, many taps", taps, dtype, flush=True)
        plan = lib.causal_conv_plan(F.CausalConvShape.packed(B, T, C, taps, K.TYPES[dtype]))
        assert plan.walks == 1
        x, state = K.Dev(lib, (B, T, C), dtype, None, rng.standard_normal((B, T, C))), K.Dev(lib, (B, taps - 1, C), dtype, None, rng.standard_normal((B, taps - 1, C)))
        w, bias = (rng.standard_normal((C, taps)) / np.sqrt(taps)).astype(np.float32), (0.3 * rng.standard_normal(C)).astype(np.float32)
        y, first = K.Dev(lib, (B, T, C), dtype), state.values
        lib.causal_conv(plan, x.ptr, K.floats(lib, w), K.floats(lib, bias), y.ptr, state.ptr, state.ptr)
        want, last, z, tz = S.causal_conv(x.values, w.astype(np.float64), bias.astype(np.float64), True, first, None)
        S.close(y.get(), want, K.ROUND[dtype] * np.abs(want) + 1.1 * tz + (8 + 2 * np.abs(z)) * K.EPS * np.abs(want) + K.TINY[dtype], "y")
        assert np.array_equal(state.get(), last)
    finally:
        lib.release(mark)


@pytest.mark.parametrize("taps", [3, 5, 8])
def test_state_over_the_one_before_in_many_walks(lib, taps):
    """However a sequence is cut, the walks read the state before it is written over."""
    rng = np.random.default_rng(taps)
    for T in (taps - 1, 9, 13, 64, 1225):
        for C in (1, 33):
            print("causal conv, state in place", taps, T, C, flush=True)
            x, given = rng.standard_normal((2, T, C)), rng.standard_normal((2, taps - 1, C))
            plan = lib.causal_conv_plan(F.CausalConvShape.packed(2, T, C, taps, K.TYPES["f32"]))
            dx, w = K.Dev(lib, (2, T, C), "f32", None, x), K.floats(lib, rng.standard_normal((C, taps)))
            apart, same = K.Dev(lib, (2, taps - 1, C), "f32", None, given), K.Dev(lib, (2, taps - 1, C), "f32", None, given)
            after, one, two = K.Dev(lib, (2, taps - 1, C), "f32"), K.Dev(lib, (2, T, C), "f32"), K.Dev(lib, (2, T, C), "f32")
            lib.causal_conv(plan, dx.ptr, w, None, one.ptr, apart.ptr, after.ptr)
            lib.causal_conv(plan, dx.ptr, w, None, two.ptr, same.ptr, same.ptr)
            assert np.array_equal(one.get(), two.get()) and np.array_equal(after.get(), same.get())
