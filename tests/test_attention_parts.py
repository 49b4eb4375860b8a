"""Linear attention on the matrix cores keeps the bits that its types have: operands in bf16 parts, none of which may get lost.

Bounds that grow with the length of the sums cannot see a missing third part of 2^-17.  Here every sum has one term (a head's tokens with a value
have one channel each, no two the same one), so that an answer is a product of three or four numbers with full mantissas and owes its error to
roundings alone.  In last places of fp32: a matrix product leaves out 2 (parts that come 24 bits late) and rounds its 6 partial sums; a decay's power,
its scale and their product 3 to 5; a state besides 3 for what it is held by, 2 where it is brought back to size and 2 a segment.  On the longest
way, through a state and the scan into an answer, that is 8 + 5 + 5 + 2*3 + 2*4 + 8 + 5 = 45: 48 allowed.  In 16-bit types what is formed between two
products has two parts, 2^-16 each time: 2^-14 allowed, and then the one rounding of the result, by half the distance to its neighbour."""
import numpy as np
import pytest

import fastconv_amd as F
import tokens as K

PLACES, INNER = 48 * K.EPS, {"f32": 48 * K.EPS, "bf16": 2.0 ** -14, "f16": 2.0 ** -14}
NAMES = ("o", "state", "dq", "dk", "dv", "dstate")

CASES = [  # T, H, Hkv, Dk, Dv
    (20, 2, 2, 64, 64),
    (100, 2, 1, 128, 128),       # two heads share a key
    (64, 2, 2, 24, 40),
    (225, 2, 2, 64, 64),         # segments
    (225, 2, 1, 96, 128),
    (130, 1, 1, 200, 256),       # two states
    (225, 2, 2, 61, 63),         # single elements
    (225, 2, 1, 32, 128),
]


def half_step(x, dtype):
    """Half the distance between neighbours of the type at x."""
    bits, least = {"f32": (24, -126), "bf16": (8, -126), "f16": (11, -14)}[dtype]
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-300))), least)
    return 0.5 * 2.0 ** (e - bits + 1)


def numbers(rng, shape, dtype):
    """Of either sign around 1, with more left for the last part than the bounds have room for: in fp32 a second part of 15 bits, of which 8 stay, and a third
    of 100 last places or more."""
    x = rng.integers(0, 1 << 23, shape, dtype=np.uint32)
    if dtype == "f32":
        x = (x & 0x0f0000) | (0x4800 + (x & 0x2f80)) | (0x38 + x % 0x10)
    return np.ldexp(((x | 0x3f800000).view(np.float32)), rng.integers(-2, 3, shape)) * rng.choice([-1.0, 1.0], shape)


def operands(T, H, Hkv, Dk, Dv, dtype, seed, dense):
    """q, k of one channel of Dk a token and v, do of one of Dv, at tokens of their own; dense: v and do have all of theirs instead."""
    rng = np.random.default_rng(seed)

    def sparse(heads, D, channels):
        x = np.zeros((1, T, heads, D))
        for h in range(heads):
            n = min(T, D, channels)
            x[0, rng.permutation(T)[:n], h, rng.permutation(channels)[:n]] = numbers(rng, n, dtype)
        return x
    both = min(Dk, Dv)
    q, k = sparse(H, Dk, both), sparse(Hkv, Dk, both)
    v, do = (numbers(rng, (1, T, h, Dv), dtype) if dense else sparse(h, Dv, both) for h in (Hkv, H))
    decay = np.array([-0.004, -0.11], np.float32)[:H]
    return [K.to_type(x, dtype)[1] for x in (q, k, v, do)] + [decay]


def formula(x, scale, backward):
    q, k, v, do, g = x
    got = K.linear_attention(q, k, v, g, scale)
    return got + (K.linear_attention_backward(do, q, k, v, g, scale) if backward else ())


def worst(got, x, scale, dtype, backward):
    """The largest error of each result in units of what it may have."""
    want = formula(x, scale, backward)
    size = formula([np.abs(a) for a in x[:4]] + [x[4]], scale, backward)
    out = {}
    for name, a, w, z in zip(NAMES, got, want, size):
        wide = name in ("state", "dstate")
        tol = (PLACES * z + half_step(w, "f32")) if wide else INNER[dtype] * z + half_step(w, dtype)
        out[name] = float((np.abs(a - w) / (tol + 1e-37)).max())
    return out


def run(L, x, T, H, Hkv, Dk, Dv, dtype, scale, backward):
    q, k, v, do = (K.Dev(L, a.shape, dtype, None, a) for a in x[:4])
    g = K.floats(L, x[4])
    plan = L.linear_attention_plan(F.LinearAttentionShape.packed(1, T, H, Hkv, Dk, Dv, K.TYPES[dtype], scale))
    ws = L.alloc(max(16, plan.ws_bytes, plan.ws_backward_bytes))
    new = lambda t: K.Dev(L, t.shape, dtype)  # noqa: E731
    state = lambda: K.Dev(L, (1, H, Dk, Dv), "f32")  # noqa: E731
    o, last, dq, dk, dv, first = K.Dev(L, (1, T, H, Dv), dtype), state(), new(q), new(k), new(v), state()
    L.linear_attention(plan, q.ptr, k.ptr, v.ptr, g, o.ptr, None, last.ptr, None, ws)
    if backward:
        L.linear_attention_backward(plan, do.ptr, q.ptr, k.ptr, v.ptr, g, dq.ptr, dk.ptr, dv.ptr, None, None, first.ptr, None, ws)
    return tuple(t.get() for t in ((o, last, dq, dk, dv, first) if backward else (o, last)))


@pytest.mark.gpu
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_no_part_is_lost(case, dtype, dense):
    T, H, Hkv, Dk, Dv = case
    scale = float(np.float32(0.3))
    with F.load(0, 1 << 28) as L:
        for seed in range(3):
            print("linear attention, parts", case, dtype, dense, seed, flush=True)
            mark = L.mark()
            x = operands(T, H, Hkv, Dk, Dv, dtype, seed, dense)
            off = worst(run(L, x, T, H, Hkv, Dk, Dv, dtype, scale, not dense), x, scale, dtype, not dense)
            print(off)
            assert max(off.values()) <= 1, off
            L.release(mark)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_no_part_of_a_carried_state_is_lost(case, dtype):
    """q alone, of one channel a token: its answers are rows of the carried state, and do's gradients columns of it."""
    T, H, Hkv, Dk, Dv = case
    rng = np.random.default_rng(9)
    with F.load(0, 1 << 28) as L:
        print("linear attention, parts of a state", case, dtype, flush=True)
        q, k, v, do, g = operands(T, H, Hkv, Dk, Dv, dtype, 4, False)
        S = numbers(rng, (1, H, Dk, Dv), "f32").astype(np.float32)
        zero = K.Dev(L, (1, T, Hkv, max(Dk, Dv)), dtype, None, np.zeros((1, T, Hkv, max(Dk, Dv))))
        dq, ddo = K.Dev(L, q.shape, dtype, None, q), K.Dev(L, do.shape, dtype, None, do)
        o, last, grad, none = K.Dev(L, do.shape, dtype), K.Dev(L, S.shape, "f32"), K.Dev(L, q.shape, dtype), K.Dev(L, zero.shape, dtype)
        plan = L.linear_attention_plan(F.LinearAttentionShape.packed(1, T, H, Hkv, Dk, Dv, K.TYPES[dtype], 1.0))
        ws, s, gp = L.alloc(max(16, plan.ws_bytes, plan.ws_backward_bytes)), K.floats(L, S), K.floats(L, g)
        L.linear_attention(plan, dq.ptr, zero.ptr, zero.ptr, gp, o.ptr, s, last.ptr, None, ws)
        L.linear_attention_backward(plan, ddo.ptr, dq.ptr, zero.ptr, zero.ptr, gp, grad.ptr, none.ptr, none.ptr, s, None, None, None, ws)
        decay = np.exp(np.arange(1, T + 1)[:, None] * g.astype(np.float64))[None, :, :, None]
        S = S.astype(np.float64)
        for name, got, want in (("o", o.get(), np.einsum("bthk,bhkv->bthv", q, S) * decay), ("dq", grad.get(), np.einsum("bthv,bhkv->bthk", do, S) * decay),
                                ("state", last.get(), S * decay[0, -1][None, :, :, None])):
            kind = "f32" if name == "state" else dtype
            off = (np.abs(got - want) / (INNER[kind] * np.abs(want) + half_step(want, kind) + 1e-37)).max()
            assert off <= 1, (name, off)


def cut(x, parts):
    """What so many bf16 parts hold of x."""
    x, rest = np.zeros_like(x), np.asarray(x, np.float64)
    for _ in range(parts):
        x = x + K.to_type(rest, "bf16")[1]
        rest = rest - K.to_type(rest, "bf16")[1]
    return x


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dense", [False, True])
def test_the_bounds_see_a_lost_part(case, dense):
    """The formula with an operand a part short passes none of the bounds that it has to do with, and passes them whole."""
    T, H, Hkv, Dk, Dv = case
    scale = float(np.float32(0.3))
    for dtype, whole in (("f32", 3), ("f16", 2)):
        x = operands(T, H, Hkv, Dk, Dv, dtype, 0, dense)
        for i, reach in enumerate((("o", "dk", "dv", "dstate"), ("o", "state", "dq", "dv"), ("o", "state", "dq", "dk"), ("dq", "dk", "dv", "dstate"))):
            if dense and i == 3:
                continue
            for parts in (whole, whole - 1):
                y = list(x)
                y[i] = cut(x[i], parts)
                got = [a if n in ("state", "dstate") else K.to_type(a, dtype)[1] for n, a in zip(NAMES, formula(y, scale, not dense))]
                off = worst(got, x, scale, dtype, not dense)
                if parts == whole:
                    assert max(off.values()) <= 1, (dtype, i, off)
                else:
                    assert all(off[n] > 1 for n in reach if n in off), (dtype, i, off)
