"""Selective scans of up to four states, whose tiles have more threads than values of B and C, over whole tiles, with B and C as columns of wider rows."""
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


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("T,dtype,G,lengths", [(32, "f32", 1, None), (33, "bf16", 2, None), (64, "f16", 1, [64, 32]), (96, "bf16", 1, [31, 96]), (288, "f32", 2, [288, 128])])
def test_whole_tiles_of_few_states(lib, N, T, dtype, G, lengths):
    rng = np.random.default_rng(N + T)
    mark = lib.mark()
    try:
        print("scan of few states", N, T, dtype, G, lengths, flush=True)
        c = scan.Case(lib, rng, 2, T, 20, N, G=G, dtype=dtype, lengths=lengths, gap=40)
        y, last = c.forward()
        w = c.want
        S.close(y.get(), w.y, K.ROUND[dtype] * np.abs(w.y) + 2 * w.ty + K.TINY[dtype], "y")
        S.close(last.get(), w.state, 2 * w.tstate + 1e-30, "state")
        grads = rng.standard_normal((c.B, c.T, c.D))
        for b, n in enumerate(w.len):
            grads[b, n:] = np.nan
        dy = K.Dev(lib, grads.shape, dtype, None, grads)
        dlast = rng.standard_normal((c.B, c.D, c.N)).astype(np.float32)
        got = c.backward(dy, dlast)
        want, tol = w.backward(np.nan_to_num(dy.values), dlast)
        for f, dev in got.items():
            kind = dtype if f in ("dx", "ddelta", "dB", "dC", "dz") else "f32"
            S.close(dev.get(), want[f], K.ROUND[kind] * np.abs(want[f]) + 2 * tol[f] + K.TINY[kind], f)
    finally:
        lib.release(mark)
