"""Group norms, rotary positions and linear attention whose outputs share elements across two axes, which are refused, and axes in other orders, which are not."""
import numpy as np
import pytest

import fastconv_amd as F
import tokens as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    L = F.load(0, 1 << 28)
    yield L
    L.close()


def refused(call):
    with pytest.raises(F.FastConvError) as e:
        call()
    assert e.value.status == -1 and "overlap" in str(e.value)


def test_group_norm(lib):
    N, P, C_, G = 3, 10, 16, 4
    p = lib.alloc(1 << 20).value
    ws = lib.alloc(1 << 20)
    for image, pixel in ((C_, C_), (P * C_ - 1, C_), (C_, N * C_ - 1), (2 * C_, 2 * C_)):
        refused(lambda: lib.group_norm(lib.group_norm_plan(F.GroupNormShape(N, P, C_, G, F.F32, F.ACT_NONE, 1e-5, P * C_, C_, image, pixel)), p, p, p, p, None, None, ws))
        refused(lambda: lib.group_norm_backward(lib.group_norm_plan(F.GroupNormShape(N, P, C_, G, F.F32, F.ACT_NONE, 1e-5, image, pixel, P * C_, C_)), p, p, p, p, p, p, p,
                                                None, None, ws))
    # pixels of all images side by side: the bits of packed ones
    rng = np.random.default_rng(0)
    x, g, b = rng.standard_normal((N, P, C_)), K.floats(lib, rng.standard_normal(C_)), K.floats(lib, rng.standard_normal(C_))
    got = []
    for image, pixel in ((P * C_, C_), (C_, N * C_)):
        dx, y = K.Dev(lib, (N, P, C_), "f32", (image, pixel, 1), x), K.Dev(lib, (N, P, C_), "f32", (image, pixel, 1))
        lib.group_norm(lib.group_norm_plan(F.GroupNormShape(N, P, C_, G, F.F32, F.ACT_NONE, 1e-5, image, pixel, image, pixel)), dx.ptr, g, b, y.ptr, None, None, ws)
        got.append(y.get())
    assert np.array_equal(*got)


def test_rotary(lib):
    B, T, H, D = 2, 4, 3, 16
    p = lib.alloc(1 << 20).value
    for batch, token, head in ((T * H * D, H * D, H * D), (H * D, H * D, D), (T * H * D - 1, H * D, D), (D, H * D, D), (T * D, D, B * T * D - 1)):
        for side in ("qo", "ko"):
            s = F.RotaryShape.packed(B, T, H, H, D, (2, 3, 3), F.BF16)
            for f, v in (("_batch", batch), ("_token", token), ("_head", head)):
                setattr(s, side + f, v)
            refused(lambda: lib.rotary(s, p, p, p, p, p, p))
    # heads outside of tokens
    rng = np.random.default_rng(1)
    x, positions = rng.standard_normal((B, T, H, D)), lib.upload_raw(rng.integers(0, 50, (B, T, 3)).astype(np.int32))
    freq = K.floats(lib, rng.uniform(0.01, 1, 8))
    got = []
    for strides in ((T * H * D, H * D, D, 1), (T * D, D, B * T * D, 1)):
        dev, out = K.Dev(lib, (B, T, H, D), "f32", strides, x), K.Dev(lib, (B, T, H, D), "f32", strides)
        s = F.RotaryShape.packed(B, T, H, 0, D, (2, 3, 3), F.F32)
        s.q_batch, s.q_token, s.q_head = strides[:3]
        s.qo_batch, s.qo_token, s.qo_head = strides[:3]
        lib.rotary(s, dev.ptr, None, positions, freq, out.ptr, None)
        got.append(out.get())
    assert np.array_equal(*got)


def test_linear_attention(lib):
    B, T, H, D = 2, 40, 3, 32
    p, ws = lib.alloc(1 << 22).value, lib.alloc(1 << 24)
    bad = ((T * H * D, H * D, H * D), (H * D, H * D, D), (T * H * D - 1, H * D, D), (D, H * D, D))
    for batch, token, head in bad:
        for side in "qkvo":
            s = F.LinearAttentionShape.packed(B, T, H, H, D, D, F.F32, 0.25)
            for f, v in (("_batch", batch), ("_token", token), ("_head", head)):
                setattr(s, side + f, v)
            plan = lib.linear_attention_plan(s)
            if side == "o":
                refused(lambda: lib.linear_attention(plan, p, p, p, p, p, ws=ws))
            else:
                refused(lambda: lib.linear_attention_backward(plan, p, p, p, p, p, p, p, p, ws=ws))
    # heads outside of tokens
    rng = np.random.default_rng(2)
    data = [rng.standard_normal((B, T, H, D)) for _ in range(3)]
    g = K.floats(lib, -rng.uniform(0.01, 0.5, H))
    got = []
    for strides in ((T * H * D, H * D, D, 1), (T * D, D, B * T * D, 1)):
        q, k, v = (K.Dev(lib, (B, T, H, D), "f32", strides, a) for a in data)
        o = K.Dev(lib, (B, T, H, D), "f32", strides)
        s = F.LinearAttentionShape.packed(B, T, H, H, D, D, F.F32, 0.25)
        for side in "qkvo":
            for f, n in zip(("_batch", "_token", "_head"), strides):
                setattr(s, side + f, n)
        lib.linear_attention(lib.linear_attention_plan(s), q.ptr, k.ptr, v.ptr, g, o.ptr, ws=ws)
        got.append(o.get())
    assert np.array_equal(*got)
