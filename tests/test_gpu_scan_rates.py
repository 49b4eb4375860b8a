"""Gradients of selective scans whose rates are minus infinity, zero and so large that nothing is left: what has decayed passes no gradient, the others' are as
elsewhere, and nothing of an infinite rate reaches a step's gradient or another state's."""
import numpy as np
import pytest

import fastconv_amd as F
import state_space as S
import test_gpu_selective_scan as scan
import tokens as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("T,lengths", [(1, None), (3, [3, 0]), (40, [40, 7]), (64, [64, 32]), (700, [700, 33])])
@pytest.mark.parametrize("N", [4, 16, 33])
def test_gradients(lib, T, lengths, gate, N):
    rng = np.random.default_rng(T + N)
    B, D = (1 if lengths is None else 2), 6
    rates = np.tile(np.resize([-np.inf, 0.0, -1e30, -2.0], N), (D, 1))
    rates[1] = np.resize([-0.5, -np.inf], N)
    mark = lib.mark()
    try:
        print("gradients of infinite rates", T, N, gate, flush=True)
        with np.errstate(invalid="ignore", over="ignore"):
            c = scan.Case(lib, rng, B, T, D, N, rates=rates, lengths=lengths, gate=gate)
            grads = rng.standard_normal((B, T, D))
            for b, n in enumerate(c.want.len):
                grads[b, n:] = np.nan
            dy, dlast = K.Dev(lib, grads.shape, "f32", None, grads), rng.standard_normal((B, D, N)).astype(np.float32)
            got = c.backward(dy, dlast)
            want, tol = c.want.backward(np.nan_to_num(dy.values), dlast)
        assert all(np.isfinite(v).all() for v in want.values()) and all(np.isfinite(v).all() for v in tol.values())
        for f, dev in got.items():
            S.close(dev.get(), want[f], K.ROUND["f32"] * np.abs(want[f]) + 2 * tol[f] + K.TINY["f32"], f)
        dead = ~np.isfinite(rates)
        assert not got["dA"].get()[dead].any()
        for b, n in enumerate(c.want.len):
            if n:
                assert not got["dstate"].get()[b][dead].any()
    finally:
        lib.release(mark)
