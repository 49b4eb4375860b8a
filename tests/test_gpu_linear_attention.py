"""Linear attention with a decay for each head, forward and backward, against the recurrence in 64 bits.

Tolerances.  With A the same sums over absolute values: an output is rounded once to its type; a term is rounded at most twice
at every token that passes (2 T last places), once in each product's sum (D) and a few times besides; in 16-bit types what is
formed between two matrix products is held in two parts of 8 bits (2^-16 of it, twice).  States are fp32: three parts of 8 bits."""
import ctypes as C

import numpy as np
import pytest

import fastconv_amd as F
import tokens as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 2 << 30)
    yield L
    L.close()


def decays(rng, H):
    g = -np.exp2(-10 * rng.random(H)).astype(np.float32)
    if H > 1:
        g[0] = 0.0             # none
    if H > 2:
        g[1] = -np.inf         # a token sees itself alone
    if H > 3:
        g[2] = -30.0
    return g


def strides_of(layout, T, H, D):
    if layout == "heads first":
        return H * T * D, D, T * D, 1
    if layout == "joined":         # a slice of a wider projection
        return T * (H * D + 24), H * D + 24, D, 1
    if layout == "odd":
        return T * (H * D + 1) + 3, H * D + 1, D, 1
    return T * H * D, H * D, D, 1


class Call:
    def __init__(self, L, B, T, H, Hkv, Dk, Dv, dtype, seed, layout="packed", lengths=None, carry=True, scale=None, decay=None):
        rng = np.random.default_rng(seed)
        self.L, self.dtype, self.B, self.T, self.H, self.Hkv, self.Dk, self.Dv = L, dtype, B, T, H, Hkv, Dk, Dv
        self.scale = float(np.float32(Dk ** -0.5 if scale is None else scale))
        st = {"q": strides_of(layout, T, H, Dk), "k": strides_of(layout, T, Hkv, Dk), "v": strides_of(layout, T, Hkv, Dv),
              "o": strides_of(layout, T, H, Dv)}
        self.st = st
        make = lambda f, h, d: K.Dev(L, (B, T, h, d), dtype, st[f], rng.standard_normal((B, T, h, d)))  # noqa: E731
        self.q, self.k, self.v, self.do = make("q", H, Dk), make("k", Hkv, Dk), make("v", Hkv, Dv), make("o", H, Dv)
        self.g = decays(rng, H) if decay is None else np.asarray(decay, np.float32)
        self.lengths = None if lengths is None else np.asarray(lengths, np.int32)
        self.state = rng.standard_normal((B, H, Dk, Dv)).astype(np.float32) if carry else None
        self.dstate = rng.standard_normal((B, H, Dk, Dv)).astype(np.float32) if carry else None
        self.shape = F.LinearAttentionShape(B, T, H, Hkv, Dk, Dv, K.TYPES[dtype], self.scale,
                                            *(st["q"][:3] + st["k"][:3] + st["v"][:3] + st["o"][:3]))
        self.plan = L.linear_attention_plan(self.shape)
        self.gp = K.floats(L, self.g)
        self.lp = None if lengths is None else L.upload_raw(self.lengths)
        self.ws = L.alloc(max(16, self.plan.ws_bytes, self.plan.ws_backward_bytes))

    def new(self, f, h, d):
        return K.Dev(self.L, (self.B, self.T, h, d), self.dtype, self.st[f])

    def states(self, values=None):
        return K.Dev(self.L, (self.B, self.H, self.Dk, self.Dv), "f32", None, values)

    def forward(self, want_state=True):
        o, out = self.new("o", self.H, self.Dv), self.states() if want_state else None
        s = None if self.state is None else self.states(self.state)
        self.L.linear_attention(self.plan, self.q.ptr, self.k.ptr, self.v.ptr, self.gp, o.ptr, s and s.ptr, out and out.ptr, self.lp, self.ws)
        return o.get(), out.get() if out else None

    def backward(self):
        dq, dk, dv = self.new("q", self.H, self.Dk), self.new("k", self.Hkv, self.Dk), self.new("v", self.Hkv, self.Dv)
        first = self.states()
        s = None if self.state is None else self.states(self.state)
        ds = None if self.dstate is None else self.states(self.dstate)
        self.L.linear_attention_backward(self.plan, self.do.ptr, self.q.ptr, self.k.ptr, self.v.ptr, self.gp, dq.ptr, dk.ptr, dv.ptr,
                                         s and s.ptr, ds and ds.ptr, first.ptr, self.lp, self.ws)
        return dq.get(), dk.get(), dv.get(), first.get()

    def check(self):
        ab = lambda x: None if x is None else np.abs(x)  # noqa: E731
        q, k, v, do = (x.values for x in (self.q, self.k, self.v, self.do))
        places = K.EPS * (2 * self.T + self.Dk + self.Dv + 64)
        inner = places + (0 if self.dtype == "f32" else 2.0 ** -14)
        got = self.forward() + self.backward()
        want = K.linear_attention(q, k, v, self.g, self.scale, self.state, self.lengths) + \
            K.linear_attention_backward(do, q, k, v, self.g, self.scale, self.state, self.dstate, self.lengths)
        size = K.linear_attention(ab(q), ab(k), ab(v), self.g, self.scale, ab(self.state), self.lengths) + \
            K.linear_attention_backward(ab(do), ab(q), ab(k), ab(v), self.g, self.scale, ab(self.state), ab(self.dstate), self.lengths)
        for name, a, w, z in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want, size):
            wide = name in ("state", "dstate")
            tol = (places + 2.0 ** -22) * z if wide else K.ROUND[self.dtype] * np.abs(w) + inner * z + K.TINY[self.dtype]
            bad = ~(np.abs(a - w) <= tol + 1e-30)
            assert not bad.any(), "%s: %d of %d off, by up to %.3g of the tolerance" % (name, bad.sum(), bad.size, np.nanmax(np.abs(a - w) / (tol + 1e-30)))
        return got


CASES = [  # B, T, H, Hkv, Dk, Dv, dtype, layout, lengths, carry
    (1, 1, 1, 1, 1, 1, "f32", "packed", None, True),
    (1, 1, 4, 4, 128, 128, "bf16", "packed", None, True),
    (3, 1, 4, 2, 64, 96, "f16", "packed", (1, 0, 1), True),
    (2, 5, 2, 1, 16, 24, "f32", "heads first", None, False),
    (2, 16, 4, 4, 64, 64, "bf16", "packed", (16, 3), True),
    (1, 17, 2, 2, 128, 128, "f32", "packed", None, True),
    (2, 31, 4, 2, 32, 32, "bf16", "joined", None, True),
    (1, 32, 2, 2, 64, 64, "f16", "packed", None, False),
    (1, 33, 3, 1, 40, 72, "f32", "odd", None, True),
    (2, 63, 2, 2, 128, 64, "bf16", "packed", (63, 62), True),
    (1, 64, 4, 4, 128, 128, "bf16", "packed", None, True),
    (1, 64, 2, 2, 13, 29, "f16", "odd", None, True),              # no size that anything divides
    (2, 65, 2, 1, 96, 256, "bf16", "packed", None, True),
    (1, 100, 4, 2, 256, 256, "f32", "packed", None, True),        # the largest heads
    (1, 100, 2, 2, 256, 128, "f16", "heads first", None, True),
    (1, 100, 2, 2, 200, 128, "bf16", "packed", None, False),
    (5, 129, 4, 2, 64, 64, "f32", "packed", (0, 129, 1, 64, 500), True),      # none, one, past the end
    (3, 200, 4, 4, 128, 128, "bf16", "packed", (-7, 128, 127), True),
    (1, 777, 2, 2, 64, 64, "bf16", "packed", None, True),
    (1, 1500, 2, 1, 32, 48, "f16", "joined", None, False),
    (2, 1225, 2, 2, 64, 96, "f32", "packed", (1225, 640), True),
    (1, 2500, 1, 1, 128, 128, "bf16", "packed", None, True),
    (64, 3, 8, 4, 128, 96, "bf16", "packed", None, True),         # many heads, few tokens: whole rows of the states
    (130, 2, 4, 4, 50, 130, "f32", "odd", None, True),
    (128, 6, 4, 2, 128, 128, "f16", "heads first", (6, 0) * 64, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_backward(lib, case):
    B, T, H, Hkv, Dk, Dv, dtype, layout, lengths, carry = case
    mark = lib.mark()
    print("linear attention", case, flush=True)
    c = Call(lib, B, T, H, Hkv, Dk, Dv, dtype, sum(case[:6]), layout, lengths, carry)
    got = c.check()
    again = c.forward() + c.backward()      # the same call, the same bits
    assert all(np.array_equal(a, b) for a, b in zip(got, again))
    if lengths is not None:      # what lies past an end is zeros, and an empty sequence hands its state on
        for b in range(B):
            n = min(max(lengths[b], 0), T)
            for t in (got[0], got[2], got[3], got[4]):
                assert not t[b, n:].any()
            if n == 0 and carry:
                assert np.array_equal(got[1][b], c.state[b]) and np.array_equal(got[5][b], c.dstate[b])
    lib.release(mark)


@pytest.mark.parametrize("dtype,T", [("bf16", 5), ("bf16", 200), ("f16", 200), ("f32", 200)])
def test_tokens_past_the_end_are_not_read(lib, dtype, T):
    """NaN and infinities in the padding of shorter sequences reach nothing."""
    mark = lib.mark()
    lengths = (T // 2, T - 1)
    c = Call(lib, 2, T, 2, 1, 32, 32, dtype, 3, "packed", lengths)
    want = c.forward() + c.backward()
    for t, v in ((c.q, np.nan), (c.k, np.inf), (c.v, np.nan), (c.do, -np.inf)):
        x = t.values.copy()
        for b in range(2):
            x[b, lengths[b]:] = v
        t.__init__(lib, t.shape, dtype, t.strides, x)
    got = c.forward() + c.backward()
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    lib.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_prompt_in_two_parts_and_then_token_by_token(lib, dtype):
    """The state carries over: parts of a prompt, then single tokens, answer as the whole does."""
    T, H, D = 150, 3, 64
    mark = lib.mark()
    whole = Call(lib, 1, T, H, H, D, D, dtype, 17, "packed", None, True)
    want, last = whole.forward()
    state = whole.states(whole.state)
    parts, es = [], 4 if dtype == "f32" else 2
    for at, n in ((0, 70), (70, 75)) + tuple((t, 1) for t in range(145, T)):
        s = F.LinearAttentionShape.packed(1, n, H, H, D, D, K.TYPES[dtype], whole.scale)
        plan, o = lib.linear_attention_plan(s), K.Dev(lib, (1, n, H, D), dtype)
        ws = lib.alloc(max(16, plan.ws_bytes))
        q, k, v = (t.ptr + at * H * D * es for t in (whole.q, whole.k, whole.v))
        lib.linear_attention(plan, q, k, v, whole.gp, o.ptr, state.ptr, state.ptr, None, ws)      # in place
        parts.append(o.get())
    got = np.concatenate(parts, axis=1)
    size, ssize = K.linear_attention(*(np.abs(t.values) for t in (whole.q, whole.k, whole.v)), whole.g, whole.scale, np.abs(whole.state))
    inner = K.EPS * (4 * T + 512) + (0 if dtype == "f32" else 2.0 ** -13)
    assert (np.abs(got - want) <= 2 * K.ROUND[dtype] * np.abs(want) + inner * size).all()
    assert (np.abs(state.get() - last) <= (K.EPS * (4 * T + 512) + 2.0 ** -21) * ssize).all()
    lib.release(mark)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [9, 100])
def test_a_later_token_reaches_no_earlier_one(lib, dtype, T):
    """NaN or an infinity in a key or value changes no answer before its token, and no other head."""
    mark = lib.mark()
    want = Call(lib, 1, T, 2, 2, 40, 72, dtype, 21).forward()[0]
    for t in (T // 2, T - 2):
        for field, value in (("k", np.nan), ("v", np.nan), ("v", np.inf), ("q", np.inf)):
            print("linear attention, not finite", dtype, T, t, field, value, flush=True)
            c = Call(lib, 1, T, 2, 2, 40, 72, dtype, 21)
            dev = getattr(c, field)
            x = dev.values.copy()
            x[0, t, 0, 3] = value
            dev.__init__(lib, dev.shape, dtype, dev.strides, x)
            got = c.forward()[0]
            assert np.array_equal(got[0, :t], want[0, :t]) and np.array_equal(got[:, :, 1], want[:, :, 1])
            assert not np.isfinite(got[0, t, 0]).all()
            lib.release(mark)
            mark = lib.mark()
    lib.release(mark)


def test_gradient_against_differences(lib):
    """Gradients along random directions against central differences of the recurrence in 64 bits."""
    mark = lib.mark()
    for T in (7, 90):
        print("linear attention, differences", T, flush=True)
        c = Call(lib, 2, T, 4, 2, 16, 24, "f32", T, "packed", (T, T - 3))
        q, k, v, w = (t.values for t in (c.q, c.k, c.v, c.do))
        s, ws = c.state.astype(np.float64), c.dstate.astype(np.float64)

        def loss(q, k, v, s):
            o, S = K.linear_attention(q, k, v, c.g, c.scale, s, c.lengths)
            return (o * w).sum() + (S * ws).sum()
        dq, dk, dv, ds = c.backward()
        rng, e = np.random.default_rng(1), 1e-3      # the loss is of third order at most: truncation of e^2
        for i, (x, d) in enumerate(((q, dq), (k, dk), (v, dv), (s, ds))):
            u = rng.standard_normal(x.shape)
            args = [q, k, v, s]
            up, down = list(args), list(args)
            up[i], down[i] = x + e * u, x - e * u
            diff = (loss(*up) - loss(*down)) / (2 * e)
            assert abs((d * u).sum() - diff) <= 2e-5 * (np.abs(d * u).sum() + 1), "qkvs"[i]
    lib.release(mark)


def test_optional_states(lib):
    mark = lib.mark()
    for T in (3, 100):
        c = Call(lib, 2, T, 2, 2, 32, 32, "bf16", 5, "packed", None, False)
        o, _ = c.forward()
        o2, none = c.forward(want_state=False)
        assert none is None and np.array_equal(o, o2)
        dq, dk, dv, _ = c.backward()
        again = c.new("q", 2, 32), c.new("k", 2, 32), c.new("v", 2, 32)
        lib.linear_attention_backward(c.plan, c.do.ptr, c.q.ptr, c.k.ptr, c.v.ptr, c.gp, *(t.ptr for t in again), ws=c.ws)
        assert all(np.array_equal(a, b.get()) for a, b in zip((dq, dk, dv), again))
    lib.release(mark)


def test_long_memory_keeps_its_decay(lib):
    """A decay's rounding must not build up over the tokens: a half-life of 7000 over 6000 of them, in fp32."""
    mark = lib.mark()
    T = 6000
    c = Call(lib, 1, T, 1, 1, 16, 16, "f32", 8, decay=[-1e-4])
    x = np.abs(c.k.values)      # of one sign, so that nothing cancels
    c.k.__init__(lib, c.k.shape, "f32", None, x)
    c.v.__init__(lib, c.v.shape, "f32", None, np.abs(c.v.values))
    o, s = c.forward()
    _, want = K.linear_attention(c.q.values, c.k.values, c.v.values, c.g, c.scale, c.state)
    assert np.linalg.norm(s - want) <= 2e-6 * np.linalg.norm(want)
    lib.release(mark)


def test_sequence_beyond_32_bits(lib):
    B, T, H, D, far = 2, 70, 1, 32, (1 << 31) + 8
    rng = np.random.default_rng(12)
    raw, q = K.to_type(rng.standard_normal((B, T, H, D)), "bf16")
    with F.load(0, 9 << 30) as L:
        big = L.alloc(2 * far + 2 * T * H * D)
        for b in range(B):
            L._check(L.c.fc_upload(L.ctx, big.value + 2 * far * b, raw[b].ctypes.data, raw[b].nbytes))
        o = K.Dev(L, (B, T, H, D), "bf16")
        s = F.LinearAttentionShape.packed(B, T, H, H, D, D, F.BF16, 0.25)
        s.q_batch = s.k_batch = s.v_batch = far
        plan, g = L.linear_attention_plan(s), np.array([-0.05], np.float32)
        L.linear_attention(plan, big, big, big, K.floats(L, g), o.ptr, ws=L.alloc(max(16, plan.ws_bytes)))
        want, _ = K.linear_attention(q, q, q, g, 0.25)
        size, _ = K.linear_attention(np.abs(q), np.abs(q), np.abs(q), g, 0.25)
        assert (np.abs(o.get() - want) <= K.ROUND["bf16"] * np.abs(want) + 2.0 ** -13 * size).all()


@pytest.mark.parametrize("T", [1, 150])
def test_replays_of_a_recorded_graph(lib, T):
    mark = lib.mark()
    c = Call(lib, 2, T, 4, 2, 64, 64, "f32", 4)
    o, out = c.new("o", 4, 64), c.states()
    dq, dk, dv, first = c.new("q", 4, 64), c.new("k", 2, 64), c.new("v", 2, 64), c.states()
    s, ds = c.states(c.state), c.states(c.dstate)

    def step():
        lib.linear_attention(c.plan, c.q.ptr, c.k.ptr, c.v.ptr, c.gp, o.ptr, s.ptr, out.ptr, None, c.ws)
        lib.linear_attention_backward(c.plan, c.do.ptr, c.q.ptr, c.k.ptr, c.v.ptr, c.gp, dq.ptr, dk.ptr, dv.ptr, s.ptr, ds.ptr, first.ptr, None, c.ws)
    lib.graph_begin()
    step()
    graph = lib.graph_end()
    outs = (o, out, dq, dk, dv, first)
    for seed in range(3):
        print("linear attention, replay", seed, flush=True)
        lib.upload_into(c.k.base, np.random.default_rng(seed).standard_normal(c.k.count))
        step()
        want = [lib.download(t.base, t.host.shape) for t in outs]
        for t in outs:
            lib.fill_zero(t.base, 4 * (t.count - 64))
        lib.graph_launch(graph)
        for t, w in zip(outs, want):
            assert np.array_equal(lib.download(t.base, t.host.shape).view(np.uint32), w.view(np.uint32))
    lib.graph_destroy(graph)
    lib.release(mark)


def test_refusals_at_the_call(lib):
    mark = lib.mark()
    plan = lib.linear_attention_plan(F.LinearAttentionShape.packed(1, 100, 4, 2, 32, 32, F.BF16))
    p = lib.alloc(4 << 20).value
    bad = F.LinearAttentionPlan.from_buffer_copy(plan)
    bad.segments += 1
    good = [p, p, p, p, p]
    for i in range(5):
        with pytest.raises(F.FastConvError) as e:
            lib.linear_attention(plan, *(None if j == i else a for j, a in enumerate(good)), ws=p)
        assert e.value.status == -1 and "fc_linear_attention" in str(e.value)
    for i in range(8):
        with pytest.raises(F.FastConvError):
            lib.linear_attention_backward(plan, *(None if j == i else p for j in range(8)), ws=p)
    for call in (lambda: lib.linear_attention(bad, *good, ws=p), lambda: lib.linear_attention(plan, p + 1, *good[1:], ws=p),
                 lambda: lib.linear_attention(plan, *good, state_in=p + 2, ws=p), lambda: lib.linear_attention(plan, *good, lengths=p + 1, ws=p),
                 lambda: lib.linear_attention_backward(plan, *([p] * 8), ws=None)):
        with pytest.raises(F.FastConvError) as e:
            call()
        assert e.value.status == -1
    lib.release(mark)


def scaled(c, fields, factor):
    """The tensors of a call times a factor, in its type."""
    for f in fields:
        t = getattr(c, f)
        t.__init__(c.L, t.shape, c.dtype, t.strides, t.values * factor)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("field", ["q", "k", "v", "do"])
def test_large_values_stay_finite_whatever_the_state_has_decayed_by(lib, dtype, field):
    """Operands of 1e35: every sum is far below the largest float, also when it is taken in by a state of which a 50000th is left."""
    mark = lib.mark()
    for T in (90, 200):      # in one piece, in segments
        print("linear attention, large", dtype, field, T, flush=True)
        c = Call(lib, 1, T, 3, 3, 64, 64, dtype, 31, decay=[-0.34, -0.05, 0.0])
        scaled(c, [field], 1e35)
        got = c.check()
        assert all(np.isfinite(x).all() for x in got)
    lib.release(mark)


@pytest.mark.parametrize("field", ["q", "k", "v", "do", "state", "dstate"])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_floats_are_numbers(lib, field, sign):
    """A value of the largest size in one place, all others small enough that every sum is a number; before its token nothing changes."""
    most, mark = float(np.finfo(np.float32).max), lib.mark()
    for T, Dk, Dv in ((20, 24, 40), (70, 64, 64), (200, 64, 128)):
        print("linear attention, largest", field, sign, T, flush=True)
        calls = []
        for value in (0.0, sign * most):
            c = Call(lib, 1, T, 3, 3, Dk, Dv, "f32", 32, decay=[-0.34, -0.05, 0.0])
            scaled(c, ["q", "k", "v", "do"], 1e-2)
            c.state *= np.float32(1e-2)
            c.dstate *= np.float32(1e-2)
            if field in ("state", "dstate"):
                getattr(c, field)[0, 1, 5, 7] = value
            else:
                t = getattr(c, field)
                x = t.values.copy()
                x[0, T // 2, 1, 7] = value
                t.__init__(lib, t.shape, "f32", t.strides, x)
            calls.append(c)
        got = calls[1].check()
        assert all(np.isfinite(x).all() for x in got)
        if field in ("q", "k", "v"):
            assert np.array_equal(got[0][0, :T // 2], calls[0].forward()[0][0, :T // 2])
    lib.release(mark)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Dk,Dv", [(30, 40), (32, 61), (60, 50), (33, 64), (20, 100), (50, 120), (100, 70), (128, 128)])
def test_single_elements_in_segments(lib, dtype, Dk, Dv):
    """Strides or sizes that no wide access fits, through every tile of the states and of the answers."""
    mark = lib.mark()
    print("linear attention, single elements", dtype, Dk, Dv, flush=True)
    c = Call(lib, 1, 225, 4, 2, Dk, Dv, dtype, Dk + Dv, "odd", None, True)
    assert c.plan.segments >= 3
    c.check()
    lib.release(mark)


@pytest.mark.parametrize("T", [4, 40])
def test_keys_shared_by_a_batch_have_no_gradient(lib, T):
    """Keys and values of one sequence may serve a whole batch; their gradients would be sums, and are refused, as are answers that overlap."""
    B, H, D = 3, 2, 32
    rng = np.random.default_rng(16)
    mark = lib.mark()
    q, o = K.Dev(lib, (B, T, H, D), "f32", None, rng.standard_normal((B, T, H, D))), K.Dev(lib, (B, T, H, D), "f32")
    k, v = (K.Dev(lib, (1, T, H, D), "f32", None, rng.standard_normal((1, T, H, D))) for _ in range(2))
    shape = F.LinearAttentionShape.packed(B, T, H, H, D, D, F.F32, 0.25)
    shape.k_batch = shape.v_batch = 0
    plan, g = lib.linear_attention_plan(shape), np.array([-0.05, -0.4], np.float32)
    ws, gp = lib.alloc(max(16, plan.ws_bytes, plan.ws_backward_bytes)), K.floats(lib, g)
    lib.linear_attention(plan, q.ptr, k.ptr, v.ptr, gp, o.ptr, ws=ws)
    both = [np.repeat(t.values, B, axis=0) for t in (k, v)]
    want, _ = K.linear_attention(q.values, *both, g, 0.25)
    size, _ = K.linear_attention(np.abs(q.values), *(np.abs(t) for t in both), g, 0.25)
    assert (np.abs(o.get() - want) <= K.EPS * (2 * T + 2 * D + 64) * size).all()
    with pytest.raises(F.FastConvError) as e:
        lib.linear_attention_backward(plan, o.ptr, q.ptr, k.ptr, v.ptr, gp, q.ptr, k.ptr, v.ptr, ws=ws)
    assert e.value.status == -1 and "overlap" in str(e.value)
    for name in ("q_batch", "q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "o_batch", "o_token", "o_head"):
        shape = F.LinearAttentionShape.packed(B, T, H, H, D, D, F.F32, 0.25)
        setattr(shape, name, D - 1)
        bad = lib.linear_attention_plan(shape)
        with pytest.raises(F.FastConvError) as e:
            if name[0] == "o":
                lib.linear_attention(bad, q.ptr, k.ptr, v.ptr, gp, o.ptr, ws=ws)
            else:
                lib.linear_attention_backward(bad, o.ptr, q.ptr, k.ptr, v.ptr, gp, q.ptr, k.ptr, v.ptr, ws=ws)
        assert e.value.status == -1 and "overlap" in str(e.value)
    lib.release(mark)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("field", ["q", "k", "v", "do"])
def test_small_values_keep_their_bits(lib, dtype, field):
    """Operands of 1e-32, whose third parts are about 1e-37, are as exact in proportion as any: what a state is held by does not push them out of range.
    By size: 32 last places in fp32 and in states, where a sum's roundings are independent of one another; the rounding of the result in bf16."""
    mark = lib.mark()
    for T in (90, 200):      # in one piece, in segments
        print("linear attention, small", dtype, field, T, flush=True)
        c = Call(lib, 1, T, 3, 3, 64, 64, dtype, 33, carry=False, decay=[-0.34, -0.05, 0.0])
        scaled(c, [field], 1e-32)
        q, k, v, do = (t.values for t in (c.q, c.k, c.v, c.do))
        want = K.linear_attention(q, k, v, c.g, c.scale) + K.linear_attention_backward(do, q, k, v, c.g, c.scale)
        for name, a, w in zip(("o", "state", "dq", "dk", "dv", "dstate"), c.forward() + c.backward(), want):
            wide = dtype == "f32" or name in ("state", "dstate")
            off = np.linalg.norm(a - w) / np.linalg.norm(w)
            assert off <= (32 * K.EPS if wide else K.ROUND[dtype]), (name, off)
    lib.release(mark)
