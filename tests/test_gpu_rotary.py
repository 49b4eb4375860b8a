"""Rotary positions with several axes against the formula in 64 bits.

Tolerance: a result is rounded once to its type; before that the angle is exact to 2^-25 of a turn's fraction (2 pi 2^-25 < 4 last
places), cosine and sine err by 4 last places, the two products and their sum by one each: 8 last places of |a| + |b|."""
import ctypes as C

import numpy as np
import pytest

import fastconv_amd as F
import tokens as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


def ladder(pairs):
    return np.concatenate([10000.0 ** (-np.arange(n) / max(n, 1)) for n in pairs]).astype(np.float32)


def check(x, got, positions, inv_freq, pairs, interleaved, inverse, dtype):
    want = K.rotary(x, positions, inv_freq, pairs, interleaved, inverse)
    size = np.abs(x).max(axis=-1, keepdims=True) * 2
    bad = np.abs(got - want) > K.ROUND[dtype] * np.abs(want) + 8 * K.EPS * size + K.TINY[dtype]
    assert not bad.any(), "%d off by up to %.3g" % (bad.sum(), np.abs(got - want).max())
    R2 = 2 * sum(pairs)
    assert np.array_equal(got[..., R2:], x[..., R2:])      # the rest passes bit by bit


CASES = [  # B, T, Hq, Hk, D, pairs, dtype, interleaved
    (1, 1, 1, 0, 2, (1,), "f32", False),
    (1, 1, 1, 1, 2, (1,), "bf16", True),
    (3, 1, 32, 8, 128, (16, 24, 24), "bf16", False),      # a token each
    (2, 35, 12, 12, 80, (0, 16, 16), "f32", True),        # part of the channels, an axis without pairs
    (2, 35, 12, 4, 80, (7, 12, 13), "f16", False),
    (1, 70, 3, 1, 65, (5, 6), "f16", True),               # odd channels
    (1, 70, 3, 1, 65, (5, 6), "bf16", False),
    (2, 1, 5, 5, 256, (32, 32, 32, 32), "bf16", True),
    (1, 1025, 2, 1, 64, (32,), "bf16", False),
    (2, 1600, 4, 2, 32, (4, 6, 6), "f16", True),          # several tokens a workgroup, the last one short
    (1, 9001, 1, 0, 36, (9, 9), "f32", False),
    (1, 3, 2, 2, 1024, (512,), "f32", False),             # the largest head
    (2, 33, 2, 1, 20, (4, 2), "f32", True),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_turns(lib, case, inverse):
    B, T, Hq, Hk, D, pairs, dtype, interleaved = case
    rng = np.random.default_rng(sum(case[:5]))
    mark = lib.mark()
    print("rotary", case, inverse, flush=True)
    q, k = K.Dev(lib, (B, T, Hq, D), dtype, None, rng.standard_normal((B, T, Hq, D))), None
    qo, ko = K.Dev(lib, (B, T, Hq, D), dtype), None
    if Hk:
        k = K.Dev(lib, (B, T, Hk, D), dtype, None, rng.standard_normal((B, T, Hk, D)))
        ko = K.Dev(lib, (B, T, Hk, D), dtype)
    positions = rng.integers(-3000, 70000, (B, T, len(pairs))).astype(np.int32)
    inv_freq = ladder(pairs)
    s = F.RotaryShape.packed(B, T, Hq, Hk, D, pairs, K.TYPES[dtype], interleaved)
    lib.rotary(s, q.ptr, k.ptr if Hk else None, lib.upload_raw(positions), K.floats(lib, inv_freq), qo.ptr, ko.ptr if Hk else None, inverse)
    check(q.values, qo.get(), positions, inv_freq, pairs, interleaved, inverse, dtype)
    if Hk:
        check(k.values, ko.get(), positions, inv_freq, pairs, interleaved, inverse, dtype)
        # in place: the same bits
        want = qo.get(), ko.get()
        p, f = lib.upload_raw(positions), K.floats(lib, inv_freq)
        lib.rotary(s, q.ptr, k.ptr, p, f, q.ptr, k.ptr, inverse)
        assert np.array_equal(q.get(), want[0]) and np.array_equal(k.get(), want[1])
    lib.release(mark)


def test_any_position_keeps_its_angle(lib):
    """The ends of int32, where a product in 32 bits has lost the angle."""
    positions = np.array([[[2 ** 31 - 1], [-2 ** 31], [16777217], [123456789], [0]]], np.int32)
    T, D = positions.shape[1], 64
    inv_freq = ladder((32,))
    inv_freq[0], inv_freq[1] = 1.0, 3.1415927
    mark = lib.mark()
    x = K.Dev(lib, (1, T, 1, D), "f32", None, np.random.default_rng(0).standard_normal((1, T, 1, D)))
    y = K.Dev(lib, (1, T, 1, D), "f32")
    lib.rotary(F.RotaryShape.packed(1, T, 1, 0, D, (32,)), x.ptr, None, lib.upload_raw(positions), K.floats(lib, inv_freq), y.ptr, None)
    check(x.values, y.get(), positions, inv_freq, (32,), False, False, "f32")
    lib.release(mark)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("odd", [0, 1])
def test_strides_and_shared_positions(lib, interleaved, odd):
    """Heads before tokens in q, a slice of a joined projection in k, outputs the other way round; odd strides."""
    B, T, Hq, Hk, D, pairs, dtype = 2, 37, 4, 2, 32, (4, 5, 7), "bf16"
    rng = np.random.default_rng(9)
    mark = lib.mark()
    qs, ks = (Hq * T * D + odd, D, T * D, 1), (T * (5 * D + odd) + 3 * odd, 5 * D + odd, D, 1)
    q = K.Dev(lib, (B, T, Hq, D), dtype, qs, rng.standard_normal((B, T, Hq, D)), odd)
    k = K.Dev(lib, (B, T, Hk, D), dtype, ks, rng.standard_normal((B, T, Hk, D)))
    qo, ko = K.Dev(lib, (B, T, Hq, D), dtype, ks[:2] + (D, 1)), K.Dev(lib, (B, T, Hk, D), dtype, (Hk * T * D, D, T * D, 1))
    positions = rng.integers(0, 300, (1, T, 3)).astype(np.int32)
    s = F.RotaryShape(B, T, Hq, Hk, D, 3, (C.c_int * 4)(*pairs), int(interleaved), F.BF16, 0, *(qs[:3] + ks[:3] + tuple(qo.strides[:3]) + tuple(ko.strides[:3])))
    inv_freq = ladder(pairs)
    lib.rotary(s, q.ptr, k.ptr, lib.upload_raw(positions), K.floats(lib, inv_freq), qo.ptr, ko.ptr)
    both = np.repeat(positions, B, axis=0)
    check(q.values, qo.get(), both, inv_freq, pairs, interleaved, False, dtype)
    check(k.values, ko.get(), both, inv_freq, pairs, interleaved, False, dtype)
    lib.release(mark)


def test_backward_is_the_transpose(lib):
    """<turn(x), y> = <x, turn back(y)>, and central differences of <turn(x), y> along a direction."""
    B, T, H, D, pairs = 2, 50, 3, 48, (6, 8, 8)
    rng = np.random.default_rng(11)
    positions, inv_freq = rng.integers(0, 2000, (B, T, 3)).astype(np.int32), ladder(pairs)
    mark = lib.mark()
    x, y = (K.Dev(lib, (B, T, H, D), "f32", None, rng.standard_normal((B, T, H, D))) for _ in range(2))
    tx, by = K.Dev(lib, (B, T, H, D), "f32"), K.Dev(lib, (B, T, H, D), "f32")
    s, p, f = F.RotaryShape.packed(B, T, H, 0, D, pairs), lib.upload_raw(positions), K.floats(lib, inv_freq)
    lib.rotary(s, x.ptr, None, p, f, tx.ptr, None)
    lib.rotary(s, y.ptr, None, p, f, by.ptr, None, True)
    a, b = (tx.get() * y.values).sum(), (x.values * by.get()).sum()
    size = np.abs(x.values * y.values).sum()
    assert abs(a - b) <= 16 * K.EPS * size * 2
    u = rng.standard_normal((B, T, H, D))
    loss = lambda v: (K.rotary(v, positions, inv_freq, pairs, False, False) * y.values).sum()  # noqa: E731
    d = (loss(x.values + 1e-3 * u) - loss(x.values - 1e-3 * u)) / 2e-3
    assert abs((by.get() * u).sum() - d) <= 16 * K.EPS * np.abs(u * np.abs(y.values)).sum() * 2
    lib.release(mark)


def test_values_that_are_not_finite_stay_in_their_pair(lib):
    x = np.random.default_rng(1).standard_normal((1, 4, 2, 32)).astype(np.float32)
    clean = x.copy()
    x[0, 1, 0, 3], x[0, 2, 1, 20], x[0, 3, 1, 31] = np.nan, np.inf, np.nan
    positions = np.arange(4, dtype=np.int32).reshape(1, 4, 1) + 1
    mark = lib.mark()
    outs = []
    for v in (x, clean):
        d, o = K.Dev(lib, v.shape, "f32", None, v), K.Dev(lib, v.shape, "f32")
        lib.rotary(F.RotaryShape.packed(1, 4, 2, 0, 32, (14,)), d.ptr, None, lib.upload_raw(positions), K.floats(lib, ladder((14,))), o.ptr, None)
        outs.append(o.get())
    touched = np.zeros(x.shape, bool)
    touched[0, 1, 0, [3, 17]] = touched[0, 2, 1, [20, 6]] = touched[0, 3, 1, 31] = True
    assert np.array_equal(outs[0][~touched], outs[1][~touched]) and not np.isfinite(outs[0][touched]).any()
    lib.release(mark)


def test_sequence_beyond_32_bits(lib):
    B, T, H, D, far = 2, 5, 2, 64, (1 << 31) + 8
    rng = np.random.default_rng(12)
    raw, values = K.to_type(rng.standard_normal((B, T, H, D)), "bf16")
    positions, inv_freq = rng.integers(0, 99, (B, T, 1)).astype(np.int32), ladder((32,))
    with F.load(0, 9 << 30) as L:
        big, y = L.alloc(2 * far + 2 * T * H * D), K.Dev(L, (B, T, H, D), "bf16")
        for b in range(B):
            L._check(L.c.fc_upload(L.ctx, big.value + 2 * far * b, raw[b].ctypes.data, raw[b].nbytes))
        s = F.RotaryShape.packed(B, T, H, 0, D, (32,), F.BF16)
        s.q_batch = far
        L.rotary(s, big, None, L.upload_raw(positions), K.floats(L, inv_freq), y.ptr, None)
        check(values, y.get(), positions, inv_freq, (32,), False, False, "bf16")


def test_replays_of_a_recorded_graph(lib):
    B, T, H, D = 2, 100, 2, 64
    mark = lib.mark()
    x, y = K.Dev(lib, (B, T, H, D), "f32", None, np.zeros((B, T, H, D))), K.Dev(lib, (B, T, H, D), "f32")
    s = F.RotaryShape.packed(B, T, H, 0, D, (16, 16))
    p, f = lib.upload_raw(np.random.default_rng(0).integers(0, 500, (B, T, 2)).astype(np.int32)), K.floats(lib, ladder((16, 16)))
    lib.graph_begin()
    lib.rotary(s, x.ptr, None, p, f, y.ptr, None)
    graph = lib.graph_end()
    for seed in range(3):
        lib.upload_into(x.base, np.random.default_rng(seed).standard_normal(x.count))
        lib.rotary(s, x.ptr, None, p, f, y.ptr, None)
        want = lib.download(y.base, y.host.shape)
        lib.fill_zero(y.base, 4 * (y.count - 64))
        lib.graph_launch(graph)
        assert np.array_equal(lib.download(y.base, y.host.shape).view(np.uint32), want.view(np.uint32))
    lib.graph_destroy(graph)
    lib.release(mark)


def test_refusals(lib):
    mark = lib.mark()
    p = lib.alloc(1 << 20).value

    def refused(status, **change):
        s = F.RotaryShape.packed(2, 8, 4, 2, 64, (8, 12, 12), F.BF16)
        args = dict(q=p, k=p, positions=p, inv_freq=p, q_out=p, k_out=p)
        for name, v in change.items():
            if name in args:
                args[name] = v
            elif name == "pairs":
                s.pairs[0] = v
            else:
                setattr(s, name, v)
        with pytest.raises(F.FastConvError) as e:
            lib.rotary(s, **args)
        assert e.value.status == status and "fc_rotary" in str(e.value), change
    for name in ("B", "T", "Hq", "D", "axes"):
        refused(-1, **{name: 0})
    refused(-1, Hk=-1)
    refused(-1, axes=5)
    refused(-1, dtype=3)
    refused(-1, pairs=-1)
    refused(-1, pairs=9)                 # 33 pairs of 64 channels
    refused(-1, q_token=-1)
    refused(-6, T=1 << 24)               # of two sequences
    for name in ("q", "k", "positions", "inv_freq", "q_out", "k_out"):
        refused(-1, **{name: None})
    refused(-1, q=p + 1)
    refused(-1, positions=p + 2)
    refused(-6, D=1026)
    refused(-6, B=2 ** 20, T=2 ** 20)
    lib.release(mark)


@pytest.mark.parametrize("B,T", [(1, 2 ** 25 - 1), (1, 2 ** 25), (31, (2 ** 25 - 1) // 31)])
def test_tokens_that_no_launch_holds_are_refused(lib, B, T):
    """Two tokens a workgroup, the last one with one of its own: 2^25 - 1 would be 2^32 threads, one more than a launch holds."""
    assert B * T >= 2 ** 25 - 1
    mark = lib.mark()
    p = lib.alloc(1 << 10).value
    with pytest.raises(F.FastConvError) as e:
        lib.rotary(F.RotaryShape.packed(B, T, 1, 0, 2, (1,)), p, None, p, p, p, None)
    assert e.value.status == -6 and "2^25 - 2" in str(e.value)
    lib.release(mark)


def test_as_many_tokens_as_a_launch_holds(lib):
    """2^25 - 2 tokens of one pair, which share the positions of 2730 sequences."""
    B, T = 2730, (2 ** 25 - 2) // 2730
    assert B * T == 2 ** 25 - 2
    rng = np.random.default_rng(13)
    raw, values = K.to_type(rng.standard_normal((T, 2)), "f16")
    mark = lib.mark()
    print("rotary, tokens", B * T, flush=True)
    positions = rng.integers(0, 5000, (1, T, 1)).astype(np.int32)
    x = lib.upload_raw(np.broadcast_to(raw, (B, T, 2)))
    s = F.RotaryShape.packed(B, T, 1, 0, 2, (1,), F.F16, shared_positions=True)
    lib.rotary(s, x, None, lib.upload_raw(positions), K.floats(lib, ladder((1,)) * np.float32(0.01)), x, None)
    got = lib.download(x, (B, T, 2), np.float16)
    assert (got == got[0]).all()
    check(values.reshape(1, T, 1, 2), got[:1].astype(np.float64).reshape(1, T, 1, 2), positions, ladder((1,)) * np.float32(0.01), (1,), False, False, "f16")
    lib.release(mark)


def test_outputs_that_share_heads_are_refused(lib):
    mark = lib.mark()
    p = lib.alloc(1 << 20).value
    for name in ("qo_batch", "qo_token", "qo_head", "ko_batch", "ko_token", "ko_head"):
        for value in (0, 63):
            s = F.RotaryShape.packed(2, 8, 4, 2, 64, (8, 12, 12), F.BF16)
            setattr(s, name, value)
            with pytest.raises(F.FastConvError) as e:
                lib.rotary(s, p, p, p, p, p, p)
            assert e.value.status == -1 and "overlap" in str(e.value)
    lib.release(mark)
