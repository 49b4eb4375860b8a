"""Causal convolutions and selective scans in layouts other than packed ones: tokens of all sequences side by side, groups outside of tokens, and outputs that
share elements, which are refused."""
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


def refused(call):
    with pytest.raises(F.FastConvError) as e:
        call()
    assert e.value.status == -1 and "overlap" in str(e.value)


def test_convolution_of_tokens_side_by_side(lib):
    """[T][B][C] gives the bits of [B][T][C], forward and backward."""
    rng = np.random.default_rng(0)
    B, T, C, taps = 3, 77, 34, 4
    x, dy = rng.standard_normal((B, T, C)), rng.standard_normal((B, T, C))
    w, space = K.floats(lib, rng.standard_normal((C, taps))), None
    got = []
    for strides in ((T * C, C, 1), (C, B * C, 1), (C + 1, B * (C + 1) + 5, 1)):
        new = lambda v=None: K.Dev(lib, (B, T, C), "f32", strides, v)  # noqa: E731
        a, up, y, dx, dw = new(x), new(dy), new(), new(), K.Dev(lib, (C, taps), "f32")
        plan = lib.causal_conv_plan(F.CausalConvShape(B, T, C, taps, F.F32, F.ACT_SILU, strides[0], strides[1], strides[0], strides[1]))
        space = lib.alloc(plan.ws_backward_bytes)
        print("convolution with strides", strides, flush=True)
        lib.causal_conv(plan, a.ptr, w, None, y.ptr)
        lib.causal_conv_backward(plan, up.ptr, a.ptr, w, None, dx.ptr, dw.ptr, ws=space)
        got.append((y.get(), dx.get(), dw.get()))
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[0], other))


def test_convolutions_whose_outputs_overlap(lib):
    B, T, C, taps = 2, 6, 8, 3
    p = [lib.alloc(1 << 16) for _ in range(5)]
    plan = lambda *strides: lib.causal_conv_plan(F.CausalConvShape(B, T, C, taps, F.F32, F.ACT_SILU, *strides))  # noqa: E731
    for batch, token in ((C, C), (T * C - 1, C), (C, B * C - 1), (4 * C, 2 * C)):
        refused(lambda: lib.causal_conv(plan(T * C, C, batch, token), p[0], p[1], None, p[2]))
        refused(lambda: lib.causal_conv_backward(plan(batch, token, T * C, C), p[0], p[1], p[2], None, p[3]))
    # one token, or one sequence: the other axis is none; rows of two sequences by turns
    for b, t, batch, token in ((1, T, C, C), (B, 1, C, C), (B, T, 3 * C, 2 * C)):
        one = lib.causal_conv_plan(F.CausalConvShape(b, t, C, taps, F.F32, F.ACT_SILU, C, C, batch, token))
        lib.causal_conv(one, p[0], p[1], None, p[2])
    lib.sync()


def scan_strides(B, T, D, G, N, order):
    if order == "packed":
        return (T * D, D), (T * G * N, G * N, N)
    if order == "side by side":
        return (D, B * D), (N, B * G * N, B * N)
    return (T * D, D), (T * N, N, B * T * N)      # groups outside


def test_scan_of_tokens_side_by_side(lib):
    rng = np.random.default_rng(1)
    B, T, D, G, N = 2, 100, 24, 2, 5
    data = {f: rng.standard_normal((B, T, D)) for f in ("x", "delta", "z", "dy")}
    data.update({f: rng.standard_normal((B, T, G, N)) for f in ("B", "C")})
    A = K.floats(lib, -np.abs(rng.standard_normal((D, N))))
    got = []
    for order in ("packed", "side by side", "groups outside"):
        wide, few = scan_strides(B, T, D, G, N, order)
        new = lambda f, v=None: K.Dev(lib, data[f].shape, "f32", (few if f in "BC" else wide) + (1,), v)  # noqa: E731
        dev = {f: new(f, v) for f, v in data.items()}
        plan = lib.selective_scan_plan(F.SelectiveScanShape(B, T, D, N, G, F.F32, 1, *wide, *wide, *wide, *few, *few, *wide))
        y, out = new("x"), {f: new(f) for f in ("x", "delta", "z", "B", "C")}
        dA = K.Dev(lib, (D, N), "f32")
        given = {f: dev[f].ptr for f in ("x", "delta", "z", "B", "C")}
        print("scan", order, flush=True)
        lib.selective_scan(plan, A=A, y=y.ptr, ws=lib.alloc(plan.ws_bytes) if plan.ws_bytes else None, **given)
        lib.selective_scan_backward(plan, dy=dev["dy"].ptr, A=A, dA=dA.ptr, ws=lib.alloc(plan.ws_backward_bytes), **{"d" + f: v.ptr for f, v in out.items()}, **given)
        got.append([y.get(), dA.get()] + [v.get() for v in out.values()])
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[0], other))


def test_scans_whose_outputs_overlap(lib):
    B, T, D, G, N = 2, 8, 16, 2, 4
    p = {f: lib.alloc(1 << 16) for f in ("x", "delta", "z", "A", "B", "C", "y", "dy", "dx", "ddelta", "dz", "dB", "dC")}
    ws = lib.alloc(1 << 24)
    wide, few = (T * D, D), (T * G * N, G * N, N)

    def plan(**change):
        s = F.SelectiveScanShape(B, T, D, N, G, F.F32, 1, *wide, *wide, *wide, *few, *few, *wide)
        for f, v in change.items():
            setattr(s, f, v)
        return lib.selective_scan_plan(s)
    given = {f: p[f] for f in ("x", "delta", "z", "A", "B", "C")}
    grads = {f: p[f] for f in ("dy", "dx", "ddelta", "dz", "dB", "dC")}
    for batch, token in ((D, D), (T * D - 1, D), (D, B * D - 1)):
        refused(lambda: lib.selective_scan(plan(y_batch=batch, y_token=token), y=p["y"], ws=ws, **given))
        for f in ("x", "delta", "z"):
            refused(lambda: lib.selective_scan_backward(plan(**{f + "_batch": batch, f + "_token": token}), ws=ws, **given, **grads))
    for batch, token, group in ((T * N, N, N), (T * G * N, N, N), (T * G * N - 1, G * N, N), (T * G * N, G * N, N - 1), (N, G * N, B * N)):
        for f in "bc":
            refused(lambda: lib.selective_scan_backward(plan(**{f + "_batch": batch, f + "_token": token, f + "_group": group}), ws=ws, **given, **grads))
