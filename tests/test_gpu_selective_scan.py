"""Selective scans, forward and backward, against the recurrence in 64 bits (bounds: state_space.Scan).

Joined segments decay by the exponential of a sum of steps, which rounds like the steps do, and add twice: their bound is twice that of the
recurrence, to which the hardware's exponential adds its last place."""
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


class Case:
    """Inputs on the device and on the host, and one call of each kind."""

    def __init__(self, L, rng, B, T, D, N, G=1, dtype="f32", gate=True, skip=True, bias=True, carry=True, lengths=None, gap=0, softplus=True, rates=None):
        self.L, self.B, self.T, self.D, self.N, self.G, self.dtype, self.gate, self.skip, self.carry = L, B, T, D, N, G, dtype, gate, skip, carry
        n = S.lengths_of(lengths, B, T)

        def sequence(v, shared=False):
            v = v.copy()
            for b in range(B):
                v[b, n[b]:] = np.nan      # not read
            row = (G * (N + gap) if shared else D + gap)
            strides = (T * row + 3 * (gap > 0), row, N + gap, 1) if shared else (T * row + 3 * (gap > 0), row, 1)
            return K.Dev(L, v.shape, dtype, strides, v)
        self.sequence = sequence
        self.x, self.delta = sequence(rng.standard_normal((B, T, D))), sequence(0.5 * rng.standard_normal((B, T, D)) if softplus else rng.uniform(0, 0.2, (B, T, D)))
        self.z = sequence(2 * rng.standard_normal((B, T, D))) if gate else None
        self.b, self.c = (sequence(rng.standard_normal((B, T, G, N)), True) for _ in range(2))
        step = np.exp(rng.uniform(np.log(1e-3), np.log(0.1), D))
        self.bias = np.log(np.expm1(step)).astype(np.float32) if bias and softplus else None
        self.A = (-(rng.uniform(0.5, 1.5, (D, N)) * np.arange(1, N + 1)) if rates is None else rates).astype(np.float32)
        self.skips = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32) if skip else None
        self.state = (0.5 * rng.standard_normal((B, D, N))).astype(np.float32) if carry else None
        self.lengths, self.softplus = lengths, softplus
        up = lambda a: None if a is None else K.floats(L, a)  # noqa: E731
        self.dA, self.dD, self.dbias, self.dstate = up(self.A), up(self.skips), up(self.bias), up(self.state)
        self.dl = L.upload_raw(np.array(lengths, np.int32)) if lengths else None
        at = lambda d: tuple(d.strides[:2])  # noqa: E731
        self.shape = F.SelectiveScanShape(B, T, D, N, G, K.TYPES[dtype], int(softplus), *at(self.x), *at(self.delta), *(at(self.z) if gate else (T * D, D)),
                                          *self.b.strides[:3], *self.c.strides[:3], T * D, D)
        self.plan = L.selective_scan_plan(self.shape)
        clean = lambda d: None if d is None else np.nan_to_num(d.values)  # noqa: E731
        f64 = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
        self.want = S.Scan(clean(self.x), clean(self.delta), f64(self.A), clean(self.b), clean(self.c), f64(self.skips), clean(self.z), f64(self.bias), softplus,
                           self.state, lengths)

    def given(self):
        return dict(x=self.x.ptr, delta=self.delta.ptr, A=self.dA, B=self.b.ptr, C=self.c.ptr, D=self.dD, z=self.z.ptr if self.gate else None,
                    delta_bias=self.dbias, lengths=self.dl)

    def forward(self, state_in=0, state_out=None):
        y = K.Dev(self.L, (self.B, self.T, self.D), self.dtype)
        last = K.Dev(self.L, (self.B, self.D, self.N), "f32") if state_out is None else None
        ws = self.L.alloc(self.plan.ws_bytes) if self.plan.ws_bytes else None
        self.L.selective_scan(self.plan, y=y.ptr, state_in=self.dstate if state_in == 0 else state_in, state_out=last.ptr if last else state_out, ws=ws, **self.given())
        return y, last

    def backward(self, dy, dlast, first=True, sums=True):
        L, like = self.L, lambda d: K.Dev(self.L, d.shape, self.dtype, d.strides)  # noqa: E731
        out = {"dx": like(self.x), "ddelta": like(self.delta), "dB": like(self.b), "dC": like(self.c)}
        if self.gate:
            out["dz"] = like(self.z)
        if sums:
            out.update({"dA": K.Dev(L, (self.D, self.N), "f32"), "dD": K.Dev(L, (self.D,), "f32"), "ddelta_bias": K.Dev(L, (self.D,), "f32")})
        if first:
            out["dstate"] = K.Dev(L, (self.B, self.D, self.N), "f32")
        named = {("dstate_in" if k == "dstate" else k): v.ptr for k, v in out.items()}
        L.selective_scan_backward(self.plan, dy=dy.ptr, state_in=self.dstate, dstate_out=None if dlast is None else K.floats(L, dlast),
                                  ws=L.alloc(self.plan.ws_backward_bytes), **named, **self.given())
        return out


CASES = [  # B, T, D, N, and what is not as usual
    (1, 1, 1, 1, dict()),
    (3, 1, 70, 16, dict(dtype="bf16")),
    (2, 1, 33, 5, dict(dtype="f16", lengths=[1, 0])),
    (2, 4, 40, 16, dict(lengths=[4, 2])),
    (2, 3, 17, 64, dict(dtype="bf16", G=1, gate=False)),
    (1, 5, 64, 16, dict()),                                      # the first with tiles
    (2, 32, 64, 16, dict(dtype="bf16")),
    (2, 33, 65, 16, dict(dtype="bf16", skip=False)),
    (1, 31, 130, 4, dict(bias=False)),
    (2, 70, 30, 3, dict(dtype="f16", gate=False, carry=False)),
    (1, 64, 96, 8, dict(dtype="bf16", G=2)),
    (2, 65, 66, 11, dict(G=3, gap=5)),
    (1, 97, 40, 32, dict(dtype="f16")),
    (1, 40, 36, 27, dict(G=2, dtype="bf16")),
    (1, 45, 21, 64, dict()),
    (1, 50, 50, 50, dict(G=5, dtype="bf16", gap=3)),
    (4, 130, 20, 16, dict(lengths=[130, 0, 1, 77])),
    (3, 200, 64, 16, dict(dtype="bf16", lengths=[32, -5, 500], gate=False)),
    (1, 700, 24, 16, dict(dtype="f32")),                         # cut into segments
    (2, 515, 40, 7, dict(dtype="bf16", G=2, lengths=[515, 130])),
    (2, 300, 18, 2, dict(lengths=[299, 257])),
    (1, 400, 12, 40, dict(dtype="f16")),
    (2, 60, 32, 16, dict(softplus=False)),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:4])) + "".join("-%s=%s" % (k, v) for k, v in c[4].items()).replace(" ", ""))
def test_forward_and_backward(lib, case):
    rng = np.random.default_rng(sum(case[:4]))
    mark = lib.mark()
    try:
        print("selective scan", case, flush=True)
        c = Case(lib, rng, *case[:4], **case[4])
        y, last = c.forward()
        w, dtype = c.want, c.dtype
        S.close(y.get(), w.y, K.ROUND[dtype] * np.abs(w.y) + 2 * w.ty + K.TINY[dtype], "y")
        S.close(last.get(), w.state, 2 * w.tstate + 1e-30, "state")
        if c.carry:      # over the state before
            again, _ = c.forward(state_out=c.dstate)
            assert np.array_equal(again.get(), y.get()) and np.array_equal(lib.download(c.dstate, last.shape), last.get().astype(np.float32))
            c.dstate = K.floats(lib, c.state)
        grads = rng.standard_normal((c.B, c.T, c.D))
        for b, n in enumerate(w.len):
            grads[b, n:] = np.nan
        dy = K.Dev(lib, grads.shape, dtype, None, grads)
        dlast = rng.standard_normal((c.B, c.D, c.N)).astype(np.float32) if c.carry else None
        got = c.backward(dy, dlast)
        want, tol = w.backward(np.nan_to_num(dy.values), dlast)
        for f, dev in got.items():
            kind = dtype if f in ("dx", "ddelta", "dB", "dC", "dz") else "f32"
            S.close(dev.get(), want[f], K.ROUND[kind] * np.abs(want[f]) + 2 * tol[f] + K.TINY[kind], f)
        # again, without what may be left out: the same bits
        for f, dev in c.backward(dy, dlast, first=False, sums=False).items():
            assert np.array_equal(dev.get(), got[f].get()), f
    finally:
        lib.release(mark)


def test_tokens_one_by_one_follow_the_prompt(lib):
    """A prompt, then single tokens and a few at once, from the state that it left."""
    rng = np.random.default_rng(11)
    for N, G in ((16, 1), (5, 2)):
        mark = lib.mark()
        B, T, D = 2, 60, 48
        c = Case(lib, rng, B, T, D, N, G, carry=False)
        y, last = c.forward()
        state, parts = K.Dev(lib, (B, D, N), "f32"), K.Dev(lib, (B, T, D), "f32")
        at = 0
        print("selective scan, token by token", N, flush=True)
        for n in (40, 1, 1, 3, 1, 9, 5):
            s = F.SelectiveScanShape.from_buffer_copy(c.shape)
            s.T = n
            plan = lib.selective_scan_plan(s)
            g = c.given()
            for f, d in (("x", c.x), ("delta", c.delta), ("z", c.z), ("B", c.b), ("C", c.c)):
                g[f] = d.ptr + at * d.strides[1] * 4
            lib.selective_scan(plan, y=parts.ptr + at * D * 4, state_in=state.ptr if at else None, state_out=state.ptr,
                               ws=lib.alloc(plan.ws_bytes) if plan.ws_bytes else None, **g)
            at += n
        assert at == T
        S.close(parts.get(), c.want.y, K.ROUND["f32"] * np.abs(c.want.y) + 2 * c.want.ty, "y")
        S.close(state.get(), c.want.state, 2 * c.want.tstate, "state")
        lib.release(mark)


def test_large_and_infinite_rates(lib):
    """A rate of minus infinity forgets, one of zero never does, one that is large leaves nothing: in single tokens, tiles and segments, and past the
    end of a sequence, where a step of 0 has to leave the state as it is."""
    rng = np.random.default_rng(12)
    for T, lengths in ((1, None), (3, [3, 0]), (40, [40, 7]), (700, [700, 33])):
        B, D, N = (1 if lengths is None else 2), 6, 4
        rates = np.tile(np.array([-np.inf, 0.0, -1e30, -2.0]), (D, 1))
        mark = lib.mark()
        print("selective scan, rates", T, flush=True)
        with np.errstate(invalid="ignore", over="ignore"):
            c = Case(lib, rng, B, T, D, N, rates=rates, lengths=lengths, gate=False)
            y, last = c.forward()
        assert np.isfinite(c.want.y).all()
        S.close(y.get(), c.want.y, K.ROUND["f32"] * np.abs(c.want.y) + 2 * c.want.ty, "y")
        S.close(last.get(), c.want.state, 2 * c.want.tstate + 1e-30, "state")
        lib.release(mark)


def test_steps_of_every_size(lib):
    """softplus from far below 0, where it is an exponential, to far above, where it is its argument, and at infinities."""
    v = np.concatenate((np.linspace(-80, 80, 321), [-np.inf, 1e4, 1e30, -1e4]))
    D = len(v)
    ones = lambda *s: K.floats(lib, np.ones(s))  # noqa: E731
    for T in (1, 8):
        x, delta = ones(1, T, D), K.floats(lib, np.tile(v, (1, T, 1)))
        bc, A = ones(1, T, 1, 1), K.floats(lib, np.zeros((D, 1)))
        y = K.Dev(lib, (1, T, D), "f32")
        plan = lib.selective_scan_plan(F.SelectiveScanShape.packed(1, T, D, 1))
        lib.selective_scan(plan, x, delta, A, bc, bc, y.ptr, ws=lib.alloc(plan.ws_bytes) if plan.ws_bytes else None)
        want = np.logaddexp(0, v)
        got = y.get()[0, 0]
        # the tiny ones: e^-80 of 2^-24 places; none is lost
        S.close(got, want, 10 * K.EPS * want, "softplus")
        S.close(y.get()[0, -1], T * want, (10 + T) * K.EPS * T * want, "sums")


def test_what_is_not_finite_stays_in_its_channel_and_time(lib):
    rng = np.random.default_rng(13)
    B, T, D, N = 1, 300, 70, 16
    c = Case(lib, rng, B, T, D, N, gate=False)
    v = c.x.values.copy()
    v[0, 100, 5] = np.nan
    c.x = K.Dev(lib, v.shape, "f32", c.x.strides, v)
    y, last = c.forward()
    bad = np.isnan(y.get())
    assert bad[0, 100:, 5].all() and not bad[0, :100].any() and not bad[0, :, [d for d in range(D) if d != 5]].any()
    assert np.isnan(last.get()[0, 5]).all() and np.isfinite(np.delete(last.get(), 5, axis=1)).all()


def test_shared_inputs_and_what_overlaps(lib):
    rng = np.random.default_rng(14)
    T, D, N = 50, 20, 8
    c = Case(lib, rng, 1, T, D, N, carry=False)
    y, _ = c.forward()
    s = F.SelectiveScanShape.from_buffer_copy(c.shape)
    s.B = 3
    for f in ("x_batch", "delta_batch", "z_batch", "b_batch", "c_batch"):
        setattr(s, f, 0)
    plan = lib.selective_scan_plan(s)
    out = K.Dev(lib, (3, T, D), "f32")
    lib.selective_scan(plan, y=out.ptr, ws=lib.alloc(plan.ws_bytes) if plan.ws_bytes else None, **c.given())
    # another number of sequences is cut differently
    S.close(out.get(), np.repeat(c.want.y, 3, axis=0), np.repeat(K.ROUND["f32"] * np.abs(c.want.y) + 2 * c.want.ty, 3, axis=0), "y")
    ws = lib.alloc(plan.ws_backward_bytes)
    like = lambda n: lib.alloc(4 * n)  # noqa: E731
    wide, few = 3 * T * D, 3 * T * N
    with pytest.raises(F.FastConvError) as e:
        lib.selective_scan_backward(plan, dy=out.ptr, dx=like(wide), ddelta=like(wide), dz=like(wide), dB=like(few), dC=like(few), ws=ws, **c.given())
    assert e.value.status == -1


def test_gradient_against_differences(lib):
    rng = np.random.default_rng(15)
    B, T, D, N, G, e = 2, 45, 10, 6, 2, 1e-5
    c = Case(lib, rng, B, T, D, N, G)
    dy = K.Dev(lib, (B, T, D), "f32", None, rng.standard_normal((B, T, D)))
    dlast = rng.standard_normal((B, D, N)).astype(np.float32)
    got = {k: v.get() for k, v in c.backward(dy, dlast).items()}
    names = ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dstate")
    at = [c.x.values, c.delta.values, c.A, c.b.values, c.c.values, c.skips, c.z.values, c.bias, c.state]
    at = [a.astype(np.float64) for a in at]
    u = [rng.standard_normal(a.shape) for a in at]

    def loss(*v):
        s = S.Scan(*v[:8], True, v[8])
        return (s.y * dy.values).sum() + (s.state * dlast).sum()
    for i, name in enumerate(names):      # each by itself, then all
        step = lambda k: [a + (k * e * d if j == i else 0) for j, (a, d) in enumerate(zip(at, u))]  # noqa: E731
        diff = (loss(*step(1)) - loss(*step(-1))) / (2 * e)
        terms = got[name] * u[i]
        # differences of e^2 times third derivatives and 1e-16/e of the loss; fp32 places of the sums on the way
        assert abs(diff - terms.sum()) <= 2e-5 * np.abs(terms).sum(), name


def test_in_a_graph(lib):
    """Both passes recorded, replayed on new values between eager calls: the same bits."""
    rng = np.random.default_rng(16)
    B, T, D, N = 1, 200, 64, 16
    plan = lib.selective_scan_plan(F.SelectiveScanShape.packed(B, T, D, N))
    assert plan.segments > 1
    wide, few = B * T * D, B * T * N
    ins = {"x": wide, "delta": wide, "A": D * N, "B": few, "C": few, "D": D, "z": wide}
    dev = {k: lib.alloc(4 * n) for k, n in ins.items()}
    dy = lib.alloc(4 * wide)
    outs = {"dx": wide, "ddelta": wide, "dA": D * N, "dB": few, "dC": few, "dD": D, "dz": wide, "ddelta_bias": D, "dstate_in": B * D * N}
    sets = [({"y": lib.alloc(4 * wide), "state_out": lib.alloc(4 * B * D * N)}, {k: lib.alloc(4 * n) for k, n in outs.items()},
             lib.alloc(plan.ws_bytes), lib.alloc(plan.ws_backward_bytes)) for _ in range(2)]

    def both(s):
        lib.selective_scan(plan, ws=s[2], **dev, **s[0])
        lib.selective_scan_backward(plan, dy=dy, ws=s[3], **dev, **s[1])
    lib.graph_begin()
    both(sets[0])
    g = lib.graph_end()
    for turn in range(3):
        for k, n in ins.items():
            lib.upload_into(dev[k], -np.abs(rng.standard_normal(n)) if k == "A" else rng.standard_normal(n))
        lib.upload_into(dy, rng.standard_normal(wide))
        print("selective scan in a graph, replay", turn, flush=True)
        both(sets[1])
        lib.graph_launch(g)
        lib.sync()
        for k, n in {"y": wide, "state_out": B * D * N}.items():
            assert np.array_equal(lib.download(sets[0][0][k], (n,)), lib.download(sets[1][0][k], (n,))), k
        for k, n in outs.items():
            assert np.array_equal(lib.download(sets[0][1][k], (n,)), lib.download(sets[1][1][k], (n,))), k
    lib.graph_destroy(g)


def test_refusals(lib):
    p = [lib.alloc(1 << 16) for _ in range(12)]
    plan = lib.selective_scan_plan(F.SelectiveScanShape.packed(1, 8, 16, 4, 1, F.BF16))
    given = dict(x=p[0], delta=p[1], A=p[2], B=p[3], C=p[4], y=p[5])
    for f in given:
        with pytest.raises(F.FastConvError) as e:
            lib.selective_scan(plan, **dict(given, **{f: None}))
        assert e.value.status == -1, f
        with pytest.raises(F.FastConvError) as e:
            lib.selective_scan(plan, **dict(given, **{f: given[f].value + 1}))
        assert e.value.status == -1, f
    for f in ("D", "z", "delta_bias", "state_in", "state_out", "lengths", "ws"):
        with pytest.raises(F.FastConvError) as e:
            lib.selective_scan(plan, **dict(given, **{f: p[6].value + 1}))
        assert e.value.status == -1, f
    other = F.SelectiveScanPlan.from_buffer_copy(plan)
    other.segments += 1
    over = F.SelectiveScanShape.packed(1, 8, 16, 4, 1, F.BF16)
    over.y_token = 15
    long = lib.selective_scan_plan(F.SelectiveScanShape.packed(1, 4096, 16, 4, 1, F.BF16))
    assert long.ws_bytes
    back = dict(dy=p[5], x=p[0], delta=p[1], A=p[2], B=p[3], C=p[4], dx=p[6], ddelta=p[7], dB=p[8], dC=p[9], ws=p[10])
    calls = [lambda: lib.selective_scan(other, **given), lambda: lib.selective_scan(lib.selective_scan_plan(over), **given),
             lambda: lib.selective_scan(long, **given), lambda: lib.selective_scan_backward(plan, **dict(back, z=p[11]))]
    calls += [lambda f=f: lib.selective_scan_backward(plan, **dict(back, **{f: None})) for f in back]
    for i, call in enumerate(calls):
        with pytest.raises(F.FastConvError) as e:
            call()
        assert e.value.status == -1, i


@pytest.mark.parametrize("case", [(1, 5201, 20, 5, dict()), (2, 5500, 8, 16, dict(dtype="bf16", lengths=[5500, 3003])), (1, 130, 64, 4, dict(dtype="f16", lengths=[97])),
                                  (3, 257, 130, 2, dict(dtype="bf16", G=2))], ids=lambda c: "-".join(map(str, c[:4])))
def test_segments_of_one_tile_and_of_several(lib, case):
    """Every tile a segment, and a join over many segments of several, the last one shorter."""
    B, T, D, N, how = case
    plan = lib.selective_scan_plan(F.SelectiveScanShape.packed(B, T, D, N, how.get("G", 1), K.TYPES[how.get("dtype", "f32")]))
    assert plan.segments == (82 if T == 5201 else 86 if T == 5500 else plan.tiles)
    test_forward_and_backward(lib, case)
