"""Gradients of the state-space operators on rows and sequences that lie more than 2^32 bytes apart: the same bits as from packed ones; and rows to 8 bits."""
import numpy as np
import pytest

import fastconv_amd as F
import tokens as K
from test_gpu_state_space_far import FAR, gather, spread

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 60 << 30)
    yield L
    L.close()


def far(L, n, size):
    """Room for n parts of so many bytes."""
    return L.alloc((n - 1) * FAR + size).value


@pytest.mark.parametrize("C", [200, 5000])
def test_norm(lib, C):
    rng, mark, e, n = np.random.default_rng(C), lib.mark(), FAR // 4, 3
    print("norm gradients of far rows", C, flush=True)
    dy, h, ds = (rng.standard_normal((n, C)).astype(np.float32) for _ in range(3))
    gamma, rstd = K.floats(lib, 1 + 0.1 * rng.standard_normal(C)), K.floats(lib, np.ones(n))
    dx, dx2, dg, dg2 = lib.alloc(4 * n * C), far(lib, n, 4 * C), lib.alloc(4 * C), lib.alloc(4 * C)
    near, wide = lib.rms_norm_plan(F.RmsNormShape.packed(n, C)), lib.rms_norm_plan(F.RmsNormShape(n, C, F.F32, 1e-5, e, e, e, e))
    lib.rms_norm_backward(near, lib.upload_raw(dy), lib.upload_raw(h), gamma, rstd, dx, dg, lib.upload_raw(ds), lib.alloc(near.ws_backward_bytes))
    lib.rms_norm_backward(wide, spread(lib, dy, n, FAR), spread(lib, h, n, FAR), gamma, rstd, dx2, dg2, spread(lib, ds, n, FAR), lib.alloc(wide.ws_backward_bytes))
    assert np.array_equal(lib.download(dx, (n, C)), gather(lib, dx2, n, FAR, (C,))) and np.array_equal(lib.download(dg, (C,)), lib.download(dg2, (C,)))
    q, q2, s, s2 = lib.alloc(n * C), far(lib, n, C), lib.alloc(4 * n), lib.alloc(4 * n)
    lib.quantize_rows(n, C, F.F32, lib.upload_raw(h), q, s)
    lib.quantize_rows(n, C, F.F32, spread(lib, h, n, FAR), q2, s2, e, FAR)
    got = np.stack([lib.download(q2 + i * FAR, (C,), np.int8) for i in range(n)])
    assert np.array_equal(lib.download(q, (n, C), np.int8), got) and np.array_equal(lib.download(s, (n,)), lib.download(s2, (n,)))
    lib.release(mark)


@pytest.mark.parametrize("T", [3, 40])
def test_convolution(lib, T):
    rng, mark, e, C, n = np.random.default_rng(T), lib.mark(), FAR // 4, 33, 3
    print("convolution gradients of far sequences", T, flush=True)
    x, dy = (rng.standard_normal((n, T, C)).astype(np.float32) for _ in range(2))
    w = K.floats(lib, rng.standard_normal((C, 4)))
    dx, dx2, dw, dw2 = lib.alloc(x.nbytes), far(lib, n, 4 * T * C), lib.alloc(16 * C), lib.alloc(16 * C)
    near, wide = lib.causal_conv_plan(F.CausalConvShape.packed(n, T, C, 4)), lib.causal_conv_plan(F.CausalConvShape(n, T, C, 4, F.F32, F.ACT_SILU, e, C, e, C))
    lib.causal_conv_backward(near, lib.upload_raw(dy), lib.upload_raw(x), w, None, dx, dw, ws=lib.alloc(near.ws_backward_bytes))
    lib.causal_conv_backward(wide, spread(lib, dy, n, FAR), spread(lib, x, n, FAR), w, None, dx2, dw2, ws=lib.alloc(wide.ws_backward_bytes))
    assert np.array_equal(lib.download(dx, x.shape), gather(lib, dx2, n, FAR, (T, C))) and np.array_equal(lib.download(dw, (C, 4)), lib.download(dw2, (C, 4)))
    lib.release(mark)


@pytest.mark.parametrize("T,N", [(1, 5), (3, 16), (40, 4), (150, 33)])
def test_scan(lib, T, N):
    """Every tensor's sequences far apart, those of B and C and all gradients among them."""
    rng, mark, e, D, n = np.random.default_rng(T), lib.mark(), FAR // 4, 70, 2
    print("scan gradients of far sequences", T, N, flush=True)
    wide = {f: rng.standard_normal((n, T, D)).astype(np.float32) for f in ("x", "delta", "z", "dy")}
    few = {f: rng.standard_normal((n, T, N)).astype(np.float32) for f in ("B", "C")}
    A = K.floats(lib, -np.abs(rng.standard_normal((D, N))))
    shapes = (F.SelectiveScanShape.packed(n, T, D, N), F.SelectiveScanShape(n, T, D, N, 1, F.F32, 1, e, D, e, D, e, D, e, N, N, e, N, N, e, D))
    got = []
    for shape, apart in zip(shapes, (False, True)):
        plan = lib.selective_scan_plan(shape)
        given = {f: spread(lib, v, n, FAR) if apart else lib.upload_raw(v) for f, v in list(wide.items()) + list(few.items())}
        size = {f: v.nbytes // n for f, v in list(wide.items()) + list(few.items())}
        out = {f: far(lib, n, size[f]) if apart else lib.alloc(n * size[f]).value for f in ("x", "delta", "z", "B", "C")}
        dA, dstate = lib.alloc(4 * D * N), lib.alloc(4 * n * D * N)
        lib.selective_scan_backward(plan, A=A, dA=dA, dstate_in=dstate, ws=lib.alloc(plan.ws_backward_bytes), **{"d" + f: p for f, p in out.items()}, **given)
        got.append([gather(lib, p, n, FAR if apart else size[f], (size[f] // 4,)) for f, p in out.items()] + [lib.download(dA, (D, N)), lib.download(dstate, (n, D, N))])
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    lib.release(mark)
