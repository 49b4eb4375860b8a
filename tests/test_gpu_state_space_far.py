"""The state-space operators on rows, tokens and sequences that lie more than 2^32 bytes apart: the same bits as from packed ones."""
import numpy as np
import pytest

import fastconv_amd as F
import tokens as K

pytestmark = pytest.mark.gpu

FAR = (1 << 32) + 4096      # bytes


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 20 << 30)
    yield L
    L.close()


def spread(L, host, n, apart):
    """n equal parts of a host array, `apart` bytes from one to the next."""
    parts = np.ascontiguousarray(host).reshape(n, -1).view(np.uint8)
    at = L.alloc((n - 1) * apart + parts.shape[1]).value
    for i in range(n):
        assert L.c.fc_upload(L.ctx, at + i * apart, parts[i].ctypes.data, parts.shape[1]) == 0
    return at


def gather(L, at, n, apart, shape):
    return np.stack([L.download(at + i * apart, shape) for i in range(n)])


def test_norm(lib):
    rng, mark, e = np.random.default_rng(0), lib.mark(), FAR // 4
    print("norm of far rows", flush=True)
    x, gamma = rng.standard_normal((3, 200)).astype(np.float32), K.floats(lib, np.ones(200))
    y, y2 = lib.alloc(2400), lib.alloc(2 * FAR + 800).value
    lib.rms_norm(lib.rms_norm_plan(F.RmsNormShape(3, 200, F.F32, 1e-5, 200, 200, 200, 200)), lib.upload_raw(x), gamma, y)
    lib.rms_norm(lib.rms_norm_plan(F.RmsNormShape(3, 200, F.F32, 1e-5, e, e, e, e)), spread(lib, x, 3, FAR), gamma, y2)
    assert np.array_equal(lib.download(y, (3, 200)), gather(lib, y2, 3, FAR, (200,)))
    lib.release(mark)


@pytest.mark.parametrize("M,N,apart", [(3, 50, FAR), (2, 3, FAR), (70, 40, 1 << 26)])
def test_product(lib, M, N, apart):
    rng, mark = np.random.default_rng(M), lib.mark()
    print("product of far rows", M, N, flush=True)
    x, w = rng.integers(-127, 128, (M, 96)).astype(np.int8), rng.integers(-127, 128, (N, 96)).astype(np.int8)
    far_w = N == 3      # the matrix's rows too
    ones, y = K.floats(lib, np.ones(max(M, N))), lib.alloc(4 * M * N)
    dw = spread(lib, w, N, apart) if far_w else lib.upload_raw(w)
    lib.int8_product(lib.int8_product_plan(F.Int8ProductShape(M, N, 96, F.F32, 96 if far_w else apart, apart if far_w else 96, N)),
                     lib.upload_raw(x) if far_w else spread(lib, x, M, apart), ones, dw, ones, y)
    assert np.array_equal(lib.download(y, (M, N)), x.astype(np.float64) @ w.astype(np.float64).T)
    lib.release(mark)


@pytest.mark.parametrize("T", [3, 40])
def test_convolution(lib, T):
    rng, mark, e, C = np.random.default_rng(T), lib.mark(), FAR // 4, 33
    print("convolution of far sequences", T, flush=True)
    x, w = rng.standard_normal((3, T, C)).astype(np.float32), K.floats(lib, rng.standard_normal((C, 4)))
    y, y2 = lib.alloc(x.nbytes), lib.alloc(2 * FAR + T * C * 4).value
    lib.causal_conv(lib.causal_conv_plan(F.CausalConvShape.packed(3, T, C, 4)), lib.upload_raw(x), w, None, y)
    lib.causal_conv(lib.causal_conv_plan(F.CausalConvShape(3, T, C, 4, F.F32, F.ACT_SILU, e, C, e, C)), spread(lib, x, 3, FAR), w, None, y2)
    assert np.array_equal(lib.download(y, x.shape), gather(lib, y2, 3, FAR, (T, C)))
    lib.release(mark)


@pytest.mark.parametrize("T", [1, 3, 40, 150])
def test_scan(lib, T):
    rng, mark, e, D, N = np.random.default_rng(T), lib.mark(), FAR // 4, 70, 5
    print("scan of far sequences", T, flush=True)
    x, b, delta = rng.standard_normal((2, T, D)).astype(np.float32), rng.standard_normal((2, T, N)).astype(np.float32), rng.standard_normal((2, T, D)).astype(np.float32)
    A, y, y2 = K.floats(lib, -np.ones((D, N))), lib.alloc(x.nbytes), lib.alloc(FAR + T * D * 4).value
    near = F.SelectiveScanShape.packed(2, T, D, N)
    far = F.SelectiveScanShape(2, T, D, N, 1, F.F32, 1, e, D, T * D, D, T * D, D, T * N, N, N, T * N, N, N, e, D)
    dd, db = lib.upload_raw(delta), lib.upload_raw(b)
    for shape, at, to in ((near, lib.upload_raw(x), y), (far, spread(lib, x, 2, FAR), y2)):
        plan = lib.selective_scan_plan(shape)
        lib.selective_scan(plan, at, dd, A, db, db, to, ws=lib.alloc(plan.ws_bytes) if plan.ws_bytes else None)
    assert np.array_equal(lib.download(y, x.shape), gather(lib, y2, 2, FAR, (T, D)))
    lib.release(mark)
