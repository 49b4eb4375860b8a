"""Products of 8-bit rows whose scales are far from 1: a large one of a token beside a small one of a channel, and the other way.

As elsewhere the sum's float, the two scales and the bias are four roundings, and the result's type the last."""
import numpy as np
import pytest

import fastconv_amd as F
import tokens as K
from test_gpu_int8_product import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


# few tokens from rows that begin on 16 bytes and anywhere, tiles of every size, reductions in parts
@pytest.mark.parametrize("M,N,K_", [(5, 48, 208), (20, 33, 129), (50, 40, 33024), (70, 90, 336), (150, 300, 131), (300, 300, 8192), (1100, 1100, 1024), (4096, 4096, 272)])
@pytest.mark.parametrize("bias", [False, True])
def test_large_and_small_scales(lib, M, N, K_, bias):
    rng = np.random.default_rng(M)
    mark = lib.mark()
    try:
        print("int8 product, scales", M, N, K_, bias, flush=True)
        x, w = rng.integers(-127, 128, (M, K_)).astype(np.int8), rng.integers(-127, 128, (N, K_)).astype(np.int8)
        # sums times the token's scale pass 3.4e38; all results are numbers, the smallest among them normal ones
        xs, ws = np.float32(10.0) ** rng.choice((33, 30, 2), M).astype(np.float32), np.float32(10.0) ** rng.choice((-8, -12, -3), N).astype(np.float32)
        check(lib, x, w, xs, ws, rng.standard_normal(N).astype(np.float32) if bias else None, "f32")
        check(lib, x, w, 1 / xs, 1 / ws, None, "f32")
        # a channel's scale that is as far away
        check(lib, x, w, np.full(M, 1e-8, np.float32), np.full(N, 1e33, np.float32), None, "f32")
    finally:
        lib.release(mark)
