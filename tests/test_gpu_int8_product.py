"""Products of 8-bit rows against whole-number sums.

The sum is exact; its float, the two scales and the bias are four roundings, and the result's type the last."""
import numpy as np
import pytest

import fastconv_amd as F
import state_space as S
import tokens as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


def held(L, values, gap, offset):
    """Rows of bytes with a gap, in a buffer of another pattern; the buffer ends with the last row."""
    rows, K_ = values.shape
    pitch = K_ + gap
    host = np.full(offset + (rows - 1) * pitch + K_, 0x7f, np.int8)
    np.lib.stride_tricks.as_strided(host[offset:], values.shape, (pitch, 1))[...] = values
    return L.upload_raw(host).value + offset


def run(L, x, w, xs, ws, bias, dtype, gap=0, offset=0, y_gap=0):
    (M, K_), N = x.shape, w.shape[0]
    y = K.Dev(L, (M, N), dtype, (N + y_gap, 1))
    plan = L.int8_product_plan(F.Int8ProductShape(M, N, K_, K.TYPES[dtype], K_ + gap, K_ + gap, N + y_gap))
    space = L.alloc(plan.ws_bytes) if plan.ws_bytes else None
    L.int8_product(plan, held(L, x, gap, offset), K.floats(L, xs), held(L, w, gap, offset), K.floats(L, ws), y.ptr,
                   None if bias is None else K.floats(L, bias), space)
    return y.get()


def check(L, x, w, xs, ws, bias, dtype, **how):
    got = run(L, x, w, xs, ws, bias, dtype, **how)
    product = (x.astype(np.float64) @ w.astype(np.float64).T) * xs.astype(np.float64)[:, None] * ws
    want = product + (0 if bias is None else bias)
    S.close(got, want, 4 * K.EPS * np.abs(product) + (K.EPS + K.ROUND[dtype]) * np.abs(want) + K.TINY[dtype], "y")


CASES = [  # M, N, K, dtype, bias, gap, offset, y_gap
    (1, 1, 1, "f32", True, 0, 0, 0),
    (1, 16, 64, "bf16", False, 0, 0, 0),
    (1, 2048, 1024, "bf16", True, 0, 0, 0),
    (3, 5, 7, "f16", True, 0, 0, 0),
    (2, 100, 333, "f32", True, 3, 1, 0),
    (16, 33, 129, "bf16", True, 0, 0, 1),
    (17, 64, 128, "f16", False, 0, 0, 0),
    (33, 96, 257, "f32", True, 0, 0, 0),
    (64, 513, 1040, "bf16", True, 0, 0, 0),
    (65, 70, 100, "f32", True, 0, 0, 0),
    (65, 130, 144, "bf16", False, 16, 16, 4),
    (100, 64, 15, "f16", True, 0, 0, 0),
    (129, 200, 771, "f32", True, 9, 3, 0),
    (200, 129, 4096, "bf16", True, 0, 0, 0),
    (300, 1000, 2064, "bf16", False, 0, 0, 0),
    (513, 255, 640, "f16", True, 0, 0, 3),
    (1225, 1000, 771, "f32", True, 9, 0, 0),
    (2050, 2048, 272, "bf16", True, 0, 0, 0),
    (4100, 4352, 400, "f16", True, 0, 0, 0),
    (4100, 4352, 403, "f32", True, 0, 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_product(lib, case):
    M, N, K_, dtype, bias, gap, offset, y_gap = case
    rng = np.random.default_rng(M + N + K_)
    mark = lib.mark()
    try:
        print("int8 product", case, flush=True)
        x, w = rng.integers(-127, 128, (M, K_)).astype(np.int8), rng.integers(-127, 128, (N, K_)).astype(np.int8)
        xs, ws = (rng.uniform(0.001, 0.02, n).astype(np.float32) for n in (M, N))
        check(lib, x, w, xs, ws, rng.standard_normal(N).astype(np.float32) if bias else None, dtype, gap=gap, offset=offset, y_gap=y_gap)
    finally:
        lib.release(mark)


@pytest.mark.parametrize("M,N", [(2, 20), (70, 40), (300, 300)])
def test_largest_sums_are_exact(lib, M, N):
    """131071 products of -128 and -128, and of -128 and 127, next to the ends of 32 bits."""
    K_ = 131071
    mark = lib.mark()
    x, w = np.full((M, K_), -128, np.int8), np.full((N, K_), -128, np.int8)
    w[1::2] = 127
    print("int8 product, largest sums", M, N, flush=True)
    check(lib, x, w, np.ones(M, np.float32), np.ones(N, np.float32), None, "f32")
    lib.release(mark)


@pytest.mark.parametrize("M,N,K_", [(5, 48, 200), (130, 140, 336), (150, 300, 131)])
def test_single_elements(lib, M, N, K_):
    """One value of x and of w at a time, through every kind of place of a tile: nothing is added to another sum."""
    rng = np.random.default_rng(K_)
    one = np.ones(max(M, N), np.float32)
    for _ in range(6):
        mark = lib.mark()
        m, n, k = rng.integers(M), rng.integers(N), rng.integers(K_)
        print("int8 product, single element", m, n, k, flush=True)
        x, w = np.zeros((M, K_), np.int8), np.zeros((N, K_), np.int8)
        x[m, k], w[n, k] = 3, -7
        got = run(lib, x, w, one[:M], one[:N], None, "f32")
        want = np.zeros((M, N))
        want[m, n] = -21
        assert np.array_equal(got, want)
        lib.release(mark)


def test_scales_that_are_not_finite_stay_in_their_row(lib):
    rng = np.random.default_rng(3)
    for M in (4, 80):
        x, w = rng.integers(-127, 128, (M, 96)).astype(np.int8), rng.integers(-127, 128, (40, 96)).astype(np.int8)
        x[1] = 0
        xs, ws = np.ones(M, np.float32), np.ones(40, np.float32)
        xs[1] = np.nan
        xs[2] = 0
        mark = lib.mark()
        print("int8 product, scale of NaN", M, flush=True)
        got = run(lib, x, w, xs, ws, None, "f32")
        lib.release(mark)
        assert np.isnan(got[1]).all() and not got[2].any()
        keep = np.array([i for i in range(M) if i != 1])
        assert np.array_equal(got[keep], (x.astype(np.float64) @ w.astype(np.float64).T)[keep] * xs[keep, None])


def test_norm_and_product_together(lib):
    """As they are used: rows normed to 8 bits, and a matrix whose rows were quantised once."""
    rng = np.random.default_rng(4)
    rows, C, N = 37, 520, 264
    x, r = (K.Dev(lib, (rows, C), "bf16", None, rng.standard_normal((rows, C))) for _ in range(2))
    w = K.Dev(lib, (N, C), "f32", None, rng.standard_normal((N, C)) / np.sqrt(C))
    gamma = (1 + 0.2 * rng.standard_normal(C)).astype(np.float32)
    q, qs, wq, wqs = lib.alloc(rows * C), lib.alloc(4 * rows), lib.alloc(N * C), lib.alloc(4 * N)
    y, total = K.Dev(lib, (rows, N), "f32"), K.Dev(lib, (rows, C), "bf16")
    print("norm and product", flush=True)
    lib.quantize_rows(N, C, F.F32, w.ptr, wq, wqs)
    lib.rms_norm_int8(lib.rms_norm_plan(F.RmsNormShape.packed(rows, C, F.BF16)), x.ptr, K.floats(lib, gamma), q, qs, r.ptr, total.ptr)
    plan = lib.int8_product_plan(F.Int8ProductShape.packed(rows, N, C, F.F32))
    lib.int8_product(plan, q, qs, wq, wqs, y.ptr, None, lib.alloc(plan.ws_bytes) if plan.ws_bytes else None)
    h, _ = S.rms_norm(total.get(), gamma.astype(np.float64), 1e-5)
    want = h @ w.values.T
    # each operand is off by at most half a step, which is the row's largest / 254, and each product by both
    step = lambda a: np.abs(a).max(axis=1, keepdims=True) / 254 * 1.001  # noqa: E731
    a, b = np.abs(h), np.abs(w.values)
    tol = step(h) * b.sum(axis=1)[None] + a.sum(axis=1)[:, None] * step(w.values).T + C * step(h) * step(w.values).T
    S.close(y.get(), want, tol, "y")
    # and as a whole the errors are of either sign
    assert np.sqrt(((y.get() - want) ** 2).mean()) <= 0.02 * np.sqrt((want ** 2).mean())


def test_in_a_graph(lib):
    rng = np.random.default_rng(9)
    for M, N, K_ in ((8, 512, 1024), (200, 300, 2000)):
        plan = lib.int8_product_plan(F.Int8ProductShape.packed(M, N, K_, F.F32))
        x, w, y, y2 = lib.alloc(M * K_), lib.upload_raw(rng.integers(-127, 128, (N, K_)).astype(np.int8)), lib.alloc(4 * M * N), lib.alloc(4 * M * N)
        xs, ws = K.floats(lib, np.ones(M)), K.floats(lib, np.ones(N))
        space, space2 = (lib.alloc(plan.ws_bytes) if plan.ws_bytes else None for _ in range(2))
        lib.graph_begin()
        lib.int8_product(plan, x, xs, w, ws, y, None, space)
        g = lib.graph_end()
        for turn in range(3):
            lib.device_copy(x, lib.upload_raw(rng.integers(-127, 128, (M, K_)).astype(np.int8)), M * K_)
            print("int8 product in a graph, replay", turn, flush=True)
            lib.int8_product(plan, x, xs, w, ws, y2, None, space2)
            lib.graph_launch(g)
            lib.sync()
            assert np.array_equal(lib.download(y, (M, N)), lib.download(y2, (M, N)))
        lib.graph_destroy(g)


def test_refusals(lib):
    p = [lib.alloc(1 << 16) for _ in range(6)]
    s = F.Int8ProductShape.packed(4, 8, 16, F.BF16)
    plan = lib.int8_product_plan(s)
    other = F.Int8ProductPlan.from_buffer_copy(plan)
    other.tile = 64 if plan.tile != 64 else 128
    narrow = lib.int8_product_plan(F.Int8ProductShape(4, 8, 16, F.BF16, 16, 16, 7))
    calls = [lambda: lib.int8_product(plan, None, p[1], p[2], p[3], p[4]), lambda: lib.int8_product(plan, p[0], None, p[2], p[3], p[4]),
             lambda: lib.int8_product(plan, p[0], p[1], None, p[3], p[4]), lambda: lib.int8_product(plan, p[0], p[1], p[2], None, p[4]),
             lambda: lib.int8_product(plan, p[0], p[1], p[2], p[3], None), lambda: lib.int8_product(plan, p[0], p[1].value + 1, p[2], p[3], p[4]),
             lambda: lib.int8_product(plan, p[0], p[1], p[2], p[3], p[4].value + 1), lambda: lib.int8_product(plan, p[0], p[1], p[2], p[3], p[4], p[5].value + 2),
             lambda: lib.int8_product(other, p[0], p[1], p[2], p[3], p[4]), lambda: lib.int8_product(narrow, p[0], p[1], p[2], p[3], p[4])]
    for i, call in enumerate(calls):
        with pytest.raises(F.FastConvError) as e:
            call()
        assert e.value.status == -1, i


@pytest.mark.parametrize("case", [  # M, N, K, gap, in parts
    (1, 40, 16, 0, False),
    (1, 8193, 48, 16, False),
    (5, 4100, 144, 0, False),            # 16 channels a workgroup
    (16, 8200, 1040, 0, False),          # 32 channels, 16 tokens
    (30, 8200, 2064, 32, False),         # 32 tokens
    (50, 8200, 1168, 0, False),          # 64 tokens
    (64, 8192, 4096, 0, False),
    (3, 70, 32784, 0, True),           # a reduction in parts
    (64, 96, 33024, 16, True),
    (3, 70, 32787, 0, True),           # the same from rows that begin anywhere
    (40, 96, 33025, 3, True),
], ids=lambda c: "-".join(map(str, c)))
def test_few_tokens(lib, case):
    M, N, K_, gap, parts = case
    rng = np.random.default_rng(M + N + K_)
    mark = lib.mark()
    try:
        print("int8 product, few tokens", case, flush=True)
        plan = lib.int8_product_plan(F.Int8ProductShape(M, N, K_, K.TYPES["bf16"], K_ + gap, K_ + gap, N))
        assert plan.tile == 0 and (plan.parts > 1) == parts and plan.ws_bytes == (4 * plan.parts * M * N if parts else 0)
        x, w = rng.integers(-127, 128, (M, K_)).astype(np.int8), rng.integers(-127, 128, (N, K_)).astype(np.int8)
        xs, ws = (rng.uniform(0.001, 0.02, n).astype(np.float32) for n in (M, N))
        check(lib, x, w, xs, ws, rng.standard_normal(N).astype(np.float32), "bf16", gap=gap)
    finally:
        lib.release(mark)


@pytest.mark.parametrize("M,N,K_", [(5, 48, 208), (64, 8192, 272), (20, 8192, 400), (16, 8192, 1040)])
def test_single_elements_of_few_tokens(lib, M, N, K_):
    """One value of x and of w at a time, in rows that begin on 16 bytes."""
    rng = np.random.default_rng(K_)
    one = np.ones(max(M, N), np.float32)
    for _ in range(8):
        mark = lib.mark()
        m, n, k = rng.integers(M), rng.integers(N), rng.integers(K_)
        print("int8 product, single element of few tokens", m, n, k, flush=True)
        x, w = np.zeros((M, K_), np.int8), np.zeros((N, K_), np.int8)
        x[m, k], w[n, k] = 3, -7
        got = run(lib, x, w, one[:M], one[:N], None, "f32")
        want = np.zeros((M, N))
        want[m, n] = -21
        assert np.array_equal(got, want)
        lib.release(mark)


@pytest.mark.parametrize("M,N,K_,tile,cut", [(64, 8192, 400, 0, False), (3, 70, 33024, 0, True), (300, 300, 8192, 64, True), (4096, 4096, 4096, 256, False)])
def test_each_way_in_a_graph(lib, M, N, K_, tile, cut):
    """Captured before anything else has run it: what a kernel needs besides its launch is no part of the capture."""
    rng = np.random.default_rng(M)
    mark = lib.mark()
    try:
        plan = lib.int8_product_plan(F.Int8ProductShape.packed(M, N, K_, F.F16))
        assert plan.tile == tile and (plan.parts > 1) == cut
        x, w, y = lib.alloc(M * K_), lib.upload_raw(rng.integers(-127, 128, (N, K_)).astype(np.int8)), K.Dev(lib, (M, N), "f16")
        xs, ws = K.floats(lib, np.full(M, 1 / 64)), K.floats(lib, np.full(N, 1 / 64))
        space = lib.alloc(plan.ws_bytes) if cut else None
        print("int8 product captured first", M, N, K_, flush=True)
        lib.graph_begin()
        lib.int8_product(plan, x, xs, w, ws, y.ptr, None, space)
        g = lib.graph_end()
        for turn in range(3):
            lib.device_copy(x, lib.upload_raw(rng.integers(-127, 128, (M, K_)).astype(np.int8)), M * K_)
            print("replay", turn, flush=True)
            lib.graph_launch(g)
            lib.sync()
            got = y.get()
            lib.int8_product(plan, x, xs, w, ws, y.ptr, None, space)
            lib.sync()
            assert np.isfinite(got).all() and got.any() and np.array_equal(got, y.get())
        lib.graph_destroy(g)
    finally:
        lib.release(mark)


@pytest.mark.parametrize("K_", [1, 3, 12, 15, 16, 17, 31, 67, 130])
@pytest.mark.parametrize("M,N", [(1, 3), (40, 50), (70, 90), (300, 200)])
def test_ends_of_rows_of_every_kind(lib, M, N, K_):
    """Rows without a gap, with one, and with one that is not 16 bytes: what lies behind a row, the next one or nothing, is no part of it."""
    rng = np.random.default_rng(M + K_)
    for gap in (0, 5, 40):
        mark = lib.mark()
        print("int8 product, ends of rows", M, N, K_, gap, flush=True)
        x, w = rng.integers(-127, 128, (M, K_)).astype(np.int8), rng.integers(-127, 128, (N, K_)).astype(np.int8)
        check(lib, x, w, np.ones(M, np.float32), np.ones(N, np.float32), None, "f32", gap=gap, offset=gap % 3)
        lib.release(mark)
