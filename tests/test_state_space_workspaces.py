"""Workspaces of the state-space operators: their size to the byte, on the CPU, and on the GPU what lies before and behind them."""
import ctypes as C

import numpy as np
import pytest

import fastconv_amd as F
import tokens as K
from fastconv_amd import capi


def plan_of(shape, name, plan):
    assert getattr(capi.load_cdll(), name)(C.byref(shape), C.byref(plan)) == 0
    return plan


def test_scan_workspaces_to_the_byte():
    """Forward: what each segment adds, and its steps.  Backward: the same of every tile, of states and of gradients, what each workgroup's channels add to dB
    and dC, and what each walk adds to dA, dD and the gradient of delta_bias."""
    for B in (1, 3, 64):
        for T in (1, 4, 5, 32, 33, 1225, 16384):
            for G, per in ((1, 1), (1, 64), (1, 65), (2, 33), (4, 512)):
                for N in (1, 4, 5, 16, 17, 33, 64):
                    D = G * per
                    p = plan_of(F.SelectiveScanShape.packed(B, T, D, N, G), "fc_selective_scan_make_plan", F.SelectiveScanPlan())
                    tiles, width = -(-T // 32), 64 if N <= 16 else 32 if N <= 32 else 16
                    blocks = G * -(-per // width)
                    assert p.ws_bytes == (4 * B * p.segments * D * (N + 1) if p.segments > 1 else 0)
                    states, steps, shared, sums = B * tiles * D * N, B * tiles * D, blocks * B * T * 2 * N, B * p.walks_backward * D * (N + 2)
                    assert p.ws_backward_bytes == 4 * (2 * states + steps + shared + sums), (B, T, G, per, N)


def test_other_workspaces_to_the_byte():
    for B, T, Cc, taps in ((1, 1, 1, 2), (3, 1225, 65, 4), (64, 45, 8193, 8), (1, 16384, 2048, 4)):
        p = plan_of(F.CausalConvShape.packed(B, T, Cc, taps), "fc_causal_conv_make_plan", F.CausalConvPlan())
        assert p.ws_backward_bytes == 4 * B * p.walks_backward * (taps + 1) * Cc
    for rows, Cc in ((1, 1), (1000, 256), (100000, 257), (5000, 8192), (12544, 40001)):
        p = plan_of(F.RmsNormShape.packed(rows, Cc), "fc_rms_norm_make_plan", F.RmsNormPlan())
        assert 1 <= p.parts <= rows and p.ws_backward_bytes == 4 * p.parts * Cc
    for M, N, Kk in ((1, 64, 65536), (300, 520, 8192), (64, 96, 33024), (4096, 4096, 4096)):
        p = plan_of(F.Int8ProductShape.packed(M, N, Kk), "fc_int8_product_make_plan", F.Int8ProductPlan())
        assert p.ws_bytes == (4 * p.parts * M * N if p.parts > 1 else 0)


GUARD = 1 << 16


class Guarded:
    """A buffer of exactly so many bytes with a pattern before and behind it."""

    def __init__(self, L, nbytes):
        self.L, self.n = L, nbytes
        self.before = np.full(nbytes + 2 * GUARD, 0xa5, np.uint8)
        self.base = L.upload_raw(self.before)
        self.ptr = self.base.value + GUARD

    def check(self, what):
        now = self.L.download(self.base, self.before.shape, np.uint8)
        assert (now[:GUARD] == 0xa5).all() and (now[GUARD + self.n:] == 0xa5).all(), "%s wrote past its workspace" % what
        assert (now[GUARD:GUARD + self.n] != 0xa5).any(), "%s did not use its workspace" % what


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 30)
    yield L
    L.close()


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,G,per,N,lengths", [(1, 5, 1, 3, 1, None), (2, 33, 2, 33, 5, [33, 7]), (3, 100, 1, 65, 16, None), (1, 700, 1, 24, 17, None),
                                                 (2, 257, 3, 20, 64, [0, 257]), (1, 2000, 1, 64, 4, None), (4, 64, 1, 130, 33, [64, 32, 1, 0])])
def test_scans_keep_to_their_workspaces(lib, B, T, G, per, N, lengths):
    rng = np.random.default_rng(T)
    mark, D = lib.mark(), G * per
    try:
        print("scan workspace", B, T, G, per, N, flush=True)
        p = lib.selective_scan_plan(F.SelectiveScanShape.packed(B, T, D, N, G))
        up = lambda *s: K.floats(lib, rng.standard_normal(s))  # noqa: E731
        given = dict(x=up(B, T, D), delta=up(B, T, D), z=up(B, T, D), B=up(B, T, G, N), C=up(B, T, G, N), A=K.floats(lib, -np.abs(rng.standard_normal((D, N)))))
        if lengths:
            given["lengths"] = lib.upload_raw(np.array(lengths, np.int32))
        if p.ws_bytes:
            ws = Guarded(lib, p.ws_bytes)
            lib.selective_scan(p, y=lib.alloc(4 * B * T * D), ws=ws.ptr, **given)
            lib.sync()
            ws.check("scan")
        ws = Guarded(lib, p.ws_backward_bytes)
        wide, few = 4 * B * T * D, 4 * B * T * G * N
        lib.selective_scan_backward(p, dy=up(B, T, D), dx=lib.alloc(wide), ddelta=lib.alloc(wide), dz=lib.alloc(wide), dB=lib.alloc(few), dC=lib.alloc(few),
                                    dA=lib.alloc(4 * D * N), dD=lib.alloc(4 * D), ddelta_bias=lib.alloc(4 * D), dstate_in=lib.alloc(4 * B * D * N), ws=ws.ptr, **given)
        lib.sync()
        ws.check("scan backward")
    finally:
        lib.release(mark)


@pytest.mark.gpu
def test_the_others_keep_to_their_workspaces(lib):
    rng = np.random.default_rng(0)
    up = lambda *s: K.floats(lib, rng.standard_normal(s))  # noqa: E731
    for B, T, Cc, taps in ((1, 1, 1, 2), (2, 77, 63, 3), (5, 1225, 8, 8), (2, 3136, 130, 4)):
        mark = lib.mark()
        print("convolution workspace", B, T, Cc, taps, flush=True)
        p = lib.causal_conv_plan(F.CausalConvShape.packed(B, T, Cc, taps))
        ws = Guarded(lib, p.ws_backward_bytes)
        lib.causal_conv_backward(p, up(B, T, Cc), up(B, T, Cc), up(Cc, taps), None, lib.alloc(4 * B * T * Cc), lib.alloc(4 * Cc * taps), lib.alloc(4 * Cc), ws=ws.ptr)
        lib.sync()
        ws.check("convolution backward")
        lib.release(mark)
    for rows, Cc in ((1, 1), (3, 7), (9001, 24), (5000, 257), (2100, 1025), (300, 4100), (40, 40001)):
        mark = lib.mark()
        print("norm workspace", rows, Cc, flush=True)
        p = lib.rms_norm_plan(F.RmsNormShape.packed(rows, Cc))
        ws = Guarded(lib, p.ws_backward_bytes)
        lib.rms_norm_backward(p, up(rows, Cc), up(rows, Cc), up(Cc), up(rows), lib.alloc(4 * rows * Cc), lib.alloc(4 * Cc), ws=ws.ptr)
        lib.sync()
        ws.check("norm backward")
        lib.release(mark)
    for M, N, Kk in ((3, 70, 32784), (40, 96, 33025), (200, 130, 4096), (300, 301, 8193)):
        mark = lib.mark()
        print("product workspace", M, N, Kk, flush=True)
        p = lib.int8_product_plan(F.Int8ProductShape.packed(M, N, Kk))
        assert p.parts > 1
        ws = Guarded(lib, p.ws_bytes)
        x, w = (lib.upload_raw(rng.integers(-127, 128, n).astype(np.int8)) for n in ((M, Kk), (N, Kk)))
        lib.int8_product(p, x, up(M), w, up(N), lib.alloc(4 * M * N), ws=ws.ptr)
        lib.sync()
        ws.check("product")
        lib.release(mark)
