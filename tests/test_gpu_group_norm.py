"""Group norm with an activation, forward and backward, against the formulas in 64 bits.

Tolerances: a result is rounded once to its type (ROUND); before that everything is fp32.  The joined statistics err by a few last
places of the group's largest value, each of the dozen operations behind them by one of its result: 32 last places of
|gamma| rstd max|x - mean| + (rstd/eps part of the mean) cover both; where the mean is many times the deviation its own last
place counts, divided by the deviation.  No slope of an activation is above 1.13, nor its own slope above 1.1."""
import math

import numpy as np
import pytest

import fastconv_amd as F
import tokens as K

pytestmark = pytest.mark.gpu

ACTS = {"none": F.ACT_NONE, "relu": F.ACT_RELU, "silu": F.ACT_SILU, "gelu": F.ACT_GELU}
EPS = 1e-5


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


def inputs(rng, N, P, C):
    x = rng.standard_normal((N, P, C)) * (0.5 + rng.random(C)) + 0.5 * rng.standard_normal(C)
    return x, (1 + 0.2 * rng.standard_normal(C)).astype(np.float32), (0.2 * rng.standard_normal(C)).astype(np.float32)


def forward(L, x, gamma, beta, N, P, C, G, dtype, act, gap=0, offset=0, stats=True):
    pixel = C + gap
    dx = K.Dev(L, (N, P, C), dtype, (P * pixel, pixel, 1), x, offset)
    dy = K.Dev(L, (N, P, C), dtype, None, None, offset)
    s = F.GroupNormShape(N, P, C, G, K.TYPES[dtype], ACTS[act], EPS, P * pixel, pixel, P * C, C)
    plan = L.group_norm_plan(s)
    m, r = (K.Dev(L, (N, G), "f32") for _ in range(2))
    ws = L.alloc(plan.ws_bytes) if plan.ws_bytes else None
    g, b = (None if a is None else K.floats(L, a) for a in (gamma, beta))
    L.group_norm(plan, dx.ptr, g, b, dy.ptr, m.ptr if stats else None, r.ptr if stats else None, ws)
    return dx, dy, plan, m, r, g, b


def close(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d off, worst %.3g of its tolerance" % (what, bad.sum(), np.nanmax(np.abs(got - want) / tol))


def bounds(x, gamma, beta, G, rstd, mean):
    """fp32 error of z: 32 last places of its largest parts, and what a last place of the mean amounts to."""
    N, P, C = x.shape
    wide = lambda a: np.repeat(a, C // G, axis=-1)[:, None, :]  # noqa: E731
    spread = np.abs(x.reshape(N, P, G, -1) - mean[:, None, :, None]).max(axis=(1, 3))
    return 32 * K.EPS * (np.abs(gamma) * wide(rstd * (spread + np.abs(mean))) + np.abs(beta))


CASES = [  # N, P, C, G, dtype, act, gap
    (1, 1, 8, 2, "f32", "none", 0),           # one pixel
    (2, 1, 64, 1, "bf16", "silu", 0),
    (3, 2, 6, 3, "f32", "silu", 0),           # groups of two channels, an access that two pixels do not fill
    (1, 196, 512, 32, "bf16", "silu", 0),
    (2, 35, 192, 32, "f16", "gelu", 24),      # groups of six channels, a gap between pixels
    (2, 35, 192, 32, "bf16", "relu", 5),      # a gap that no wide access fits
    (3, 77, 63, 7, "f16", "silu", 0),         # odd channels
    (2, 130, 64, 32, "bf16", "silu", 0),
    (1, 1000, 40, 8, "f32", "gelu", 8),
    (5, 33, 24, 24, "f16", "none", 0),        # instance norm
    (2, 9, 4096, 1, "bf16", "silu", 0),       # the largest group
    (1, 5, 4097 * 2, 4097, "f32", "relu", 0),
    (2, 6, 4100, 2, "bf16", "none", 0),       # wide groups that no two share a workgroup
    (1, 3, 2051 * 3, 3, "f16", "none", 0),
    (1, 9000, 16, 4, "bf16", "silu", 0),      # many chunks
    (2, 50176, 8, 4, "f32", "silu", 0),
    (70, 5, 32, 8, "f32", "gelu", 0),         # many images
    (33, 1225, 96, 32, "bf16", "gelu", 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(lib, case):
    N, P, C, G, dtype, act, gap = case
    rng = np.random.default_rng(sum(case[:4]))
    x, gamma, beta = inputs(rng, N, P, C)
    mark = lib.mark()
    try:
        print("group norm", case, flush=True)
        dx, dy, plan, m, r, g, b = forward(lib, x, gamma, beta, N, P, C, G, dtype, act, gap)
        x = dx.values
        y, mean, rstd, xhat, z = K.group_norm(x, gamma, beta, G, EPS, act)
        tz = bounds(x, gamma, beta, G, rstd, mean)
        got = dy.get()
        close(got, y, K.ROUND[dtype] * np.abs(y) + 1.2 * tz + K.TINY[dtype], "y")
        spread = np.abs(x).reshape(N, -1).max(axis=1)[:, None]
        close(m.get(), mean, 16 * K.EPS * spread + 1e-30, "mean")
        close(r.get(), rstd, 32 * K.EPS * rstd * (1 + rstd ** 2 * spread ** 2 * K.EPS), "rstd")
        # without statistics, the same bits
        _, plain, *_ = forward(lib, x, gamma, beta, N, P, C, G, dtype, act, gap, stats=False)
        assert np.array_equal(plain.get(), got)

        grad = K.Dev(lib, (N, P, C), dtype, None, rng.standard_normal((N, P, C)))
        out = K.Dev(lib, (N, P, C), dtype, dx.strides)
        dgamma, dbeta = K.Dev(lib, (C,), "f32"), K.Dev(lib, (C,), "f32")
        ws = lib.alloc(max(4, plan.ws_backward_bytes))
        lib.group_norm_backward(plan, grad.ptr, dx.ptr, g, b, m.ptr, r.ptr, out.ptr, dgamma.ptr, dbeta.ptr, ws)
        want, wg, wb, dz = K.group_norm_backward(grad.values, x, gamma, beta, G, EPS, act)
        # dz errs with z (by the slope's slope) and by a few places of its own; the sums by 2 sqrt of their length at most times that
        tdz = np.abs(grad.values) * (1.2 * tz + 8 * K.EPS)
        if act == "relu":      # where z is within its error of the jump either slope will do
            tdz = tdz + np.abs(grad.values) * (np.abs(z) <= tz)
        txh = 32 * K.EPS * (np.abs(xhat) + np.repeat(rstd * (np.abs(mean) + spread), C // G, axis=-1)[:, None, :])
        places = K.EPS * (16 + 2 * np.sqrt(N * P))
        close(dbeta.get(), wb, tdz.sum(axis=(0, 1)) + places * np.abs(dz).sum(axis=(0, 1)) + 1e-30, "dbeta")
        close(dgamma.get(), wg, (tdz * np.abs(xhat) + np.abs(dz) * txh).sum(axis=(0, 1)) + places * np.abs(dz * xhat).sum(axis=(0, 1)) + 1e-30,
              "dgamma")
        grouped = lambda a: np.repeat(a.reshape(N, P, G, -1).mean(axis=(1, 3)), C // G, axis=-1)[:, None, :]  # noqa: E731
        rw = np.repeat(rstd, C // G, axis=-1)[:, None, :]
        ga = np.abs(gamma)
        h, th = ga * np.abs(dz), ga * tdz
        ax = np.abs(xhat)
        s1, s2 = grouped(h), grouped(h * ax)
        ts1, ts2 = grouped(th), grouped(th * ax + h * txh)
        tol = rw * (th + ts1 + ax * ts2 + txh * s2 + 2 * places * (h + s1 + ax * s2)) + 32 * K.EPS * np.abs(want)
        close(out.get(), want, K.ROUND[dtype] * np.abs(want) + tol + K.TINY[dtype], "dx")
        # again: the same bits; and without the sums
        again, only = K.Dev(lib, (N, P, C), dtype, dx.strides), K.Dev(lib, (C,), "f32")
        lib.group_norm_backward(plan, grad.ptr, dx.ptr, g, b, m.ptr, r.ptr, again.ptr, only.ptr, None, ws)
        assert np.array_equal(again.get(), out.get()) and np.array_equal(only.get(), dgamma.get())
    finally:
        lib.release(mark)


def test_gradient_against_differences(lib):
    """dx, dgamma and dbeta along random directions against central differences of the forward formula in 64 bits."""
    N, P, C, G = 2, 30, 24, 4
    rng = np.random.default_rng(5)
    for act in ("none", "silu", "gelu"):
        x, gamma, beta = inputs(rng, N, P, C)
        mark = lib.mark()
        print("group norm, differences", act, flush=True)
        dx, dy, plan, m, r, g, b = forward(lib, x, gamma, beta, N, P, C, G, "f32", act)
        x = dx.values
        w = K.Dev(lib, (N, P, C), "f32", None, rng.standard_normal((N, P, C)))
        out, dgamma, dbeta = K.Dev(lib, (N, P, C), "f32"), K.Dev(lib, (C,), "f32"), K.Dev(lib, (C,), "f32")
        lib.group_norm_backward(plan, w.ptr, dx.ptr, g, b, m.ptr, r.ptr, out.ptr, dgamma.ptr, dbeta.ptr, lib.alloc(plan.ws_backward_bytes))
        loss = lambda a, c, d: (K.group_norm(a, c, d, G, EPS, act)[0] * w.values).sum()  # noqa: E731
        e = 1e-4      # truncation is of e^2 times a third derivative of some tens
        u, ug, ub = rng.standard_normal((N, P, C)), rng.standard_normal(C), rng.standard_normal(C)
        gamma, beta = gamma.astype(np.float64), beta.astype(np.float64)
        for got, d in (((out.get() * u).sum(), (loss(x + e * u, gamma, beta) - loss(x - e * u, gamma, beta)) / (2 * e)),
                       ((dgamma.get() * ug).sum(), (loss(x, gamma + e * ug, beta) - loss(x, gamma - e * ug, beta)) / (2 * e)),
                       ((dbeta.get() * ub).sum(), (loss(x, gamma, beta + e * ub) - loss(x, gamma, beta - e * ub)) / (2 * e))):
            assert abs(got - d) <= 1e-4 * (1 + abs(d)), act
        lib.release(mark)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_mean_far_above_the_deviation(lib, dtype):
    """Values of 1000 +- 1: the variance comes from differences, not from squares."""
    N, P, C, G = 2, 700, 16, 2
    rng = np.random.default_rng(1)
    x = 1000 + rng.standard_normal((N, P, C)) * (8 if dtype == "bf16" else 1)
    x[0, 0] = 900      # and the first pixel is no typical one
    mark = lib.mark()
    dx, dy, *_ = forward(lib, x, None, None, N, P, C, G, dtype, "none")
    y, mean, rstd, *_ = K.group_norm(dx.values, 1.0, 0.0, G, EPS, "none")
    close(dy.get(), y, K.ROUND[dtype] * np.abs(y) + bounds(dx.values, np.ones(C), np.zeros(C), G, rstd, mean), "y")
    lib.release(mark)


def test_constant_groups_and_values_that_are_not_finite(lib):
    N, P, C, G = 2, 40, 32, 4
    rng = np.random.default_rng(2)
    x, gamma, beta = inputs(rng, N, P, C)
    x[0, :, 8:16] = 3.0
    x[1, 7, 3], x[1, 9, 30] = np.nan, np.inf
    mark = lib.mark()
    dx, dy, *_ = forward(lib, x, gamma, beta, N, P, C, G, "f32", "none")
    got = dy.get()
    assert np.array_equal(got[0, :, 8:16], np.broadcast_to(beta[8:16].astype(np.float64), (P, 8)))
    for n, c in ((1, slice(0, 8)), (1, slice(24, 32))):      # its own group and no other
        assert np.isnan(got[n, :, c]).all()
    clean = x.copy()
    clean[1, 7, 3] = clean[1, 9, 30] = 0
    _, ref, *_ = forward(lib, clean, gamma, beta, N, P, C, G, "f32", "none")
    assert np.array_equal(got[0], ref.get()[0]) and np.array_equal(got[1, :, 8:24], ref.get()[1, :, 8:24])
    lib.release(mark)


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_tensors_that_begin_anywhere(lib, offset):
    rng = np.random.default_rng(3)
    x, gamma, beta = inputs(rng, 2, 50, 64)
    mark = lib.mark()
    _, a, *_ = forward(lib, x, gamma, beta, 2, 50, 64, 8, "bf16", "silu", gap=8)
    _, b, *_ = forward(lib, x, gamma, beta, 2, 50, 64, 8, "bf16", "silu", gap=8, offset=offset)
    # narrower accesses join in another order
    assert np.abs(a.get() - b.get()).max() <= 2 * K.ROUND["bf16"] * np.abs(a.get()).max()
    lib.release(mark)


def test_in_place(lib):
    rng = np.random.default_rng(4)
    for N, P, C, G in ((2, 300, 64, 8), (1, 20000, 64, 8)):
        x, gamma, beta = inputs(rng, N, P, C)
        mark = lib.mark()
        _, want, *_ = forward(lib, x, gamma, beta, N, P, C, G, "f16", "silu")
        t = K.Dev(lib, (N, P, C), "f16", None, x)
        plan = lib.group_norm_plan(F.GroupNormShape.packed(N, P, C, G, F.F16, F.ACT_SILU, EPS))
        lib.group_norm(plan, t.ptr, K.floats(lib, gamma), K.floats(lib, beta), t.ptr, ws=lib.alloc(max(4, plan.ws_bytes)))
        assert np.array_equal(t.get(), want.get())
        lib.release(mark)


def test_image_beyond_32_bits(lib):
    """The second image begins 2^31 elements after the first."""
    N, P, C, G, far = 2, 40, 32, 8, (1 << 31) + 64
    rng = np.random.default_rng(6)
    x, gamma, beta = inputs(rng, N, P, C)
    raw, values = K.to_type(x, "bf16")
    with F.load(0, 9 << 30) as L:
        big, y = L.alloc(2 * far + 2 * P * C), K.Dev(L, (N, P, C), "bf16")
        for n in range(N):
            L._check(L.c.fc_upload(L.ctx, big.value + 2 * far * n, raw[n].ctypes.data, raw[n].nbytes))
        plan = L.group_norm_plan(F.GroupNormShape(N, P, C, G, F.BF16, F.ACT_SILU, EPS, far, C, P * C, C))
        ws = L.alloc(max(4, plan.ws_bytes))
        L.group_norm(plan, big, K.floats(L, gamma), K.floats(L, beta), y.ptr, ws=ws)
        want, mean, rstd, *_ = K.group_norm(values, gamma, beta, G, EPS, "silu")
        close(y.get(), want, K.ROUND["bf16"] * np.abs(want) + 1.2 * bounds(values, gamma, beta, G, rstd, mean), "y")


def test_replays_of_a_recorded_graph(lib):
    N, P, C, G = 4, 500, 64, 8
    mark = lib.mark()
    rng = np.random.default_rng(8)
    x, gamma, beta = inputs(rng, N, P, C)
    dx, dy, plan, m, r, g, b = forward(lib, x, gamma, beta, N, P, C, G, "f32", "silu")
    ws = lib.alloc(max(4, plan.ws_bytes, plan.ws_backward_bytes))
    out, dgamma, dbeta = K.Dev(lib, (N, P, C), "f32"), K.Dev(lib, (C,), "f32"), K.Dev(lib, (C,), "f32")

    def step():
        lib.group_norm(plan, dx.ptr, g, b, dy.ptr, m.ptr, r.ptr, ws)
        lib.group_norm_backward(plan, dy.ptr, dx.ptr, g, b, m.ptr, r.ptr, out.ptr, dgamma.ptr, dbeta.ptr, ws)
    lib.graph_begin()
    step()
    graph = lib.graph_end()
    for seed in range(3):
        print("group norm, replay", seed, flush=True)
        lib.upload_into(dx.base, np.concatenate([np.random.default_rng(seed).standard_normal((N * P * C,)), np.zeros(64)]))
        step()
        want = [lib.download(t.base, t.host.shape) for t in (dy, out, dgamma, dbeta)]
        for t in (dy, out, dgamma, dbeta):
            lib.fill_zero(t.base, 4 * t.count)
        lib.graph_launch(graph)
        for t, w in zip((dy, out, dgamma, dbeta), want):
            n = t.count - 64
            assert np.array_equal(lib.download(t.base, t.host.shape)[:n], w[:n])
    lib.graph_destroy(graph)
    lib.release(mark)


def test_refusals_at_the_call(lib):
    mark = lib.mark()
    plan = lib.group_norm_plan(F.GroupNormShape.packed(2, 30000, 16, 4, F.BF16))
    buf = lib.alloc(4 << 20)
    p = buf.value
    bad = F.GroupNormPlan.from_buffer_copy(plan)
    bad.chunks += 1
    for call in (lambda: lib.group_norm(bad, p, None, None, p, None, None, p),
                 lambda: lib.group_norm(plan, None, None, None, p, None, None, p),
                 lambda: lib.group_norm(plan, p, None, None, None, None, None, p),
                 lambda: lib.group_norm(plan, p, None, None, p, p, None, p),         # one statistic of two
                 lambda: lib.group_norm(plan, p, None, None, p, None, None, None),   # no workspace
                 lambda: lib.group_norm(plan, p + 1, None, None, p, None, None, p),
                 lambda: lib.group_norm(plan, p, p + 2, None, p, None, None, p),
                 lambda: lib.group_norm_backward(plan, p, p, None, None, None, p, p, None, None, p),
                 lambda: lib.group_norm_backward(plan, p, p, None, None, p, p, p, None, None, None)):
        with pytest.raises(F.FastConvError) as e:
            call()
        assert e.value.status == -1 and "fc_group_norm" in str(e.value)
    lib.release(mark)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G", [1, 32])
def test_activations_are_exact_in_proportion(lib, act, dtype, G):
    """gamma is 0, so that z is beta to the last bit, and one pixel makes dbeta the slope.

    SiLU in fp32: exp errs through its argument's rounding by 11 last places at |z| = 12, the sum, the reciprocal and the product by one each,
    16 allowed; 1 - s in the slope by half a last place of 1, times z.  GELU: exp(-z^2/2) takes over the roundings of its argument, z^2 last
    places together, 2 z^2 allowed beside 32 for all else.  In 16 bits the cheap form of erf besides: 1.5e-7."""
    C_ = 1024
    z = np.linspace(-12, 12, C_).astype(np.float32)
    rng = np.random.default_rng(7)
    mark = lib.mark()
    print("group norm, activations", act, dtype, G, flush=True)
    x = rng.standard_normal((1, 1, C_))
    dx, dy, plan, m, r, g, b = forward(lib, x, np.zeros(C_, np.float32), z, 1, 1, C_, G, dtype, act)
    grad = K.Dev(lib, (1, 1, C_), dtype, None, np.ones((1, 1, C_)))
    out, dbeta = K.Dev(lib, (1, 1, C_), dtype), K.Dev(lib, (C_,), "f32")
    lib.group_norm_backward(plan, grad.ptr, dx.ptr, g, b, m.ptr, r.ptr, out.ptr, None, dbeta.ptr, lib.alloc(max(4, plan.ws_backward_bytes)))
    z = z.astype(np.float64)
    if act == "silu":
        s, flat = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))      # and 1 - s
        y, slope, size = z * s, s + z * s * flat, s + np.abs(z) * s * flat
        ty, ts = 16 * K.EPS * np.abs(y), K.EPS * (16 * size + np.abs(z) * s)
        more = 2 * np.abs(z) * K.EPS * size
    else:
        half = 0.5 * np.array([math.erfc(-v / math.sqrt(2)) for v in z])
        bell = np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        y, slope, size = z * half, half + z * bell, half + np.abs(z) * bell
        ty, ts = (32 + 2 * z * z) * K.EPS * np.abs(y), (32 + 2 * z * z) * K.EPS * size
        more = 1.5e-7 + 4 * z * z * K.EPS * size
    if dtype != "f32":
        ty, ts = ty + more * np.abs(z), ts + more
    close(dy.get()[0, 0], y, K.ROUND[dtype] * np.abs(y) + ty + K.TINY[dtype], "y")
    close(dbeta.get(), slope, ts + 1e-37, "slope")
    lib.release(mark)


def pixels_a_thread(plan, span):
    """What a resident kernel of 1024 threads holds, rounded up to the kernels there are."""
    s = plan.shape
    cols = span // (4 if s.dtype == F.F32 else 8)
    need = -(-s.P // (1024 // cols))
    return 1 << (need - 1).bit_length()


RESIDENT = [  # N, P, C, G, dtype, act, pixels a thread forward, backward (0: two passes)
    (2, 3136, 64, 4, "f32", "silu", 16, 0),
    (1, 4096, 32, 2, "f32", "gelu", 16, 0),            # every slot taken
    (2, 2049, 64, 2, "bf16", "silu", 16, 0),
    (1, 3136, 64, 2, "f16", "gelu", 16, 0),
    (2, 2047, 96, 2, "bf16", "gelu", 16, 0),           # groups of 48: no butterflies
    (1, 2500, 48, 2, "f32", "none", 16, 0),
    (1, 1900, 48, 1, "f16", "relu", 16, 0),
    (2, 2000, 64, 4, "f32", "gelu", 8, 8),
    (2, 1025, 64, 2, "bf16", "silu", 8, 8),
    (1, 2048, 64, 2, "bf16", "gelu", 8, 8),
    (2, 1600, 64, 2, "f16", "gelu", 8, 8),
    (1, 1360, 96, 2, "f16", "silu", 8, 8),
    (2, 1300, 48, 1, "bf16", "gelu", 8, 8),
    (1, 1111, 72, 3, "f32", "silu", 8, 8),
]


@pytest.mark.parametrize("case", RESIDENT, ids=lambda c: "-".join(map(str, c)))
def test_as_many_pixels_as_a_thread_holds(lib, case):
    N, P, C_, G, dtype, act, ahead, back = case
    plan = lib.group_norm_plan(F.GroupNormShape(N, P, C_, G, K.TYPES[dtype], ACTS[act], EPS, P * C_, C_, P * C_, C_))
    assert plan.resident and pixels_a_thread(plan, plan.resident) == ahead
    assert pixels_a_thread(plan, plan.resident_backward) == back if back else plan.resident_backward == 0
    test_forward_and_backward(lib, (N, P, C_, G, dtype, act, 0))


@pytest.mark.parametrize("dtype,N,act", [("bf16", 21, "silu"), ("f16", 21, "none"), ("f32", 12, "silu")])
def test_tensors_beyond_the_last_cache(lib, dtype, N, act):
    """More than 256 MB with their result, which is then stored past the caches: three images over and over, all equal to the bit to those
    three, which are checked."""
    P, C_, G, kinds = 224 * 224, 64, 32, 3
    assert 2 * N * P * C_ * np.dtype(K.storage(dtype)).itemsize > 256 << 20
    rng = np.random.default_rng(14)
    print("group norm, beyond the cache", dtype, flush=True)
    x, gamma, beta = inputs(rng, kinds, P, C_)
    mark = lib.mark()
    plan = lib.group_norm_plan(F.GroupNormShape.packed(N, P, C_, G, K.TYPES[dtype], ACTS[act], EPS))
    assert plan.resident == 0 and plan.resident_backward == 0
    which = np.arange(N) % kinds
    raw, x = K.to_type(x, dtype)
    raw_dy, dy = K.to_type(rng.standard_normal(x.shape), dtype)
    at_x, at_dy = lib.upload_raw(raw[which]), lib.upload_raw(raw_dy[which])
    at_y, at_dx = lib.alloc(N * raw[0].nbytes), lib.alloc(N * raw[0].nbytes)
    m, r, dgamma, dbeta = (K.Dev(lib, n, "f32") for n in ((N, G), (N, G), (C_,), (C_,)))
    ws, g, b = lib.alloc(max(4, plan.ws_bytes, plan.ws_backward_bytes)), K.floats(lib, gamma), K.floats(lib, beta)
    lib.group_norm(plan, at_x, g, b, at_y, m.ptr, r.ptr, ws)
    lib.group_norm_backward(plan, at_dy, at_x, g, b, m.ptr, r.ptr, at_dx, dgamma.ptr, dbeta.ptr, ws)
    results = []
    for at in (at_y, at_dx):
        got = lib.download(at, (N, P, C_), K.storage(dtype))
        words = got.view(np.uint32 if dtype == "f32" else np.uint16)
        assert all(np.array_equal(words[n], words[n % kinds]) for n in range(N))
        results.append(K.from_type(got[:kinds], dtype))
    y, mean, rstd, xhat, z = K.group_norm(x, gamma, beta, G, EPS, act)
    tz = bounds(x, gamma, beta, G, rstd, mean)
    close(results[0], y, K.ROUND[dtype] * np.abs(y) + 1.2 * tz + K.TINY[dtype], "y")
    want, _, _, dz = K.group_norm_backward(dy, x, gamma, beta, G, EPS, act)
    # as in test_forward_and_backward
    spread = np.abs(x).reshape(kinds, -1).max(axis=1)[:, None]
    tdz = np.abs(dy) * (1.2 * tz + 8 * K.EPS)
    txh = 32 * K.EPS * (np.abs(xhat) + np.repeat(rstd * (np.abs(mean) + spread), C_ // G, axis=-1)[:, None, :])
    places = K.EPS * (16 + 2 * np.sqrt(N * P))
    grouped = lambda a: np.repeat(a.reshape(kinds, P, G, -1).mean(axis=(1, 3)), C_ // G, axis=-1)[:, None, :]  # noqa: E731
    rw, ga, ax = np.repeat(rstd, C_ // G, axis=-1)[:, None, :], np.abs(gamma), np.abs(xhat)
    h, th = ga * np.abs(dz), ga * tdz
    s1, s2 = grouped(h), grouped(h * ax)
    tol = rw * (th + grouped(th) + ax * grouped(th * ax + h * txh) + txh * s2 + 2 * places * (h + s1 + ax * s2)) + 32 * K.EPS * np.abs(want)
    close(results[1], want, K.ROUND[dtype] * np.abs(want) + tol + K.TINY[dtype], "dx")
    times = np.bincount(which, minlength=kinds).astype(np.float64)
    total = lambda a: (a.sum(axis=1) * times[:, None]).sum(axis=0)  # noqa: E731
    close(dbeta.get(), total(dz), total(tdz) + places * total(np.abs(dz)) + 1e-30, "dbeta")
    close(dgamma.get(), total(dz * xhat), total(tdz * ax + np.abs(dz) * txh) + places * total(np.abs(dz) * ax) + 1e-30, "dgamma")
    lib.release(mark)


def test_outputs_that_share_pixels_are_refused(lib):
    """One image for all of a batch is an input like any other, but no output, and its gradient would be a sum."""
    N, P, C_, G = 3, 20, 32, 4
    rng = np.random.default_rng(15)
    x, gamma, beta = inputs(rng, 1, P, C_)
    mark = lib.mark()
    dx, y = K.Dev(lib, (1, P, C_), "f32", None, x), K.Dev(lib, (N, P, C_), "f32")
    m, r = (K.Dev(lib, (N, G), "f32") for _ in range(2))
    plan = lib.group_norm_plan(F.GroupNormShape(N, P, C_, G, F.F32, F.ACT_SILU, EPS, 0, C_, P * C_, C_))
    g, b, ws = K.floats(lib, gamma), K.floats(lib, beta), lib.alloc(max(4, plan.ws_bytes, plan.ws_backward_bytes))
    lib.group_norm(plan, dx.ptr, g, b, y.ptr, m.ptr, r.ptr, ws)
    got = y.get()
    want, mean, rstd, *_ = K.group_norm(dx.values, gamma, beta, G, EPS, "silu")
    close(got[:1], want, K.ROUND["f32"] * np.abs(want) + 1.2 * bounds(dx.values, gamma, beta, G, rstd, mean), "y")
    assert np.array_equal(got[1:], got[:-1])
    with pytest.raises(F.FastConvError) as e:
        lib.group_norm_backward(plan, y.ptr, dx.ptr, g, b, m.ptr, r.ptr, dx.ptr, None, None, ws)
    assert e.value.status == -1 and "overlap" in str(e.value)
    for strides in ((P * C_, C_, 0, C_), (P * C_, C_, P * C_, C_ - 1), (P * C_, C_, P * C_, 0)):
        bad = lib.group_norm_plan(F.GroupNormShape(N, P, C_, G, F.F32, F.ACT_SILU, EPS, *strides))
        with pytest.raises(F.FastConvError) as e:
            lib.group_norm(bad, y.ptr, g, b, y.ptr, None, None, ws)
        assert e.value.status == -1 and "overlap" in str(e.value)
    lib.release(mark)
