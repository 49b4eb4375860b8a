"""The operators on tokens in 64 bits, and host arrays in the types that they take."""
import math

import numpy as np

import fastconv_amd as F

TYPES = {"f32": F.F32, "bf16": F.BF16, "f16": F.F16}
# half a last place, of a value rounded once
ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}
EPS = 2.0 ** -24


def to_type(x, dtype):
    """A float array in memory format, and the values it then stands for."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x, x.astype(np.float64)
    if dtype == "f16":
        y = x.astype(np.float16)
        return y, y.astype(np.float64)
    bits = x.view(np.uint32)
    y = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    y = np.where(np.isnan(x), np.uint16(0x7fc0), y)
    return y, from_type(y, dtype)


def from_type(y, dtype):
    if dtype == "bf16":
        return (y.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return y.astype(np.float64)


def storage(dtype):
    return {"f32": np.float32, "bf16": np.uint16, "f16": np.float16}[dtype]


class Dev:
    """A tensor on the device with strides in elements, in a buffer filled with a pattern before and after."""

    def __init__(self, L, shape, dtype, strides=None, values=None, offset=0):
        self.L, self.shape, self.dtype = L, tuple(shape), dtype
        es = np.dtype(storage(dtype)).itemsize
        packed = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        self.strides = packed if strides is None else list(strides)
        self.count = offset + sum((n - 1) * s for n, s in zip(shape, self.strides)) + 1 + 64
        self.offset = offset
        self.host = np.full(self.count * es, 0x5a, np.uint8).view(storage(dtype))
        self.values = None
        if values is not None:
            raw, self.values = to_type(values, dtype)
            self._view(self.host)[...] = raw.reshape(self.shape)
        self.base = L.upload_raw(self.host)
        self.ptr = self.base.value + offset * es

    def _view(self, flat):
        es = flat.dtype.itemsize
        return np.lib.stride_tricks.as_strided(flat[self.offset:], self.shape, [s * es for s in self.strides])

    def get(self):
        """The values on the device; whatever lies between them is as it was."""
        now = self.L.download(self.base, self.host.shape, self.host.dtype)
        got = self._view(now).copy()
        untouched = now.copy()
        self._view(untouched)[...] = self._view(self.host)
        assert untouched.tobytes() == self.host.tobytes(), "elements outside the tensor were written"
        return from_type(got, self.dtype)


def floats(L, x):
    return L.upload_raw(np.ascontiguousarray(x, np.float32))


# ---------------------------------------------------------------- group norm

def erf(x):
    return np.vectorize(math.erf, otypes=[np.float64])(x)


def activation(z, act):
    if act == "relu":
        return np.maximum(z, 0)
    if act == "silu":
        return z / (1 + np.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + erf(z / math.sqrt(2)))
    return z


def activation_slope(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "silu":
        s = 1 / (1 + np.exp(-z))
        return s + z * s * (1 - s)
    if act == "gelu":
        return 0.5 * (1 + erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return np.ones_like(z)


def group_norm(x, gamma, beta, G, eps, act):
    N, P, C = x.shape
    xg = x.reshape(N, P, G, C // G)
    mean = xg.mean(axis=(1, 3))
    var = ((xg - mean[:, None, :, None]) ** 2).mean(axis=(1, 3))
    rstd = 1 / np.sqrt(var + eps)
    xhat = ((xg - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(N, P, C)
    z = xhat * gamma + beta
    return activation(z, act), mean, rstd, xhat, z


def group_norm_backward(dy, x, gamma, beta, G, eps, act):
    N, P, C = x.shape
    _, _, rstd, xhat, z = group_norm(x, gamma, beta, G, eps, act)
    dz = dy * activation_slope(z, act)
    h = (dz * gamma).reshape(N, P, G, C // G)
    xg = xhat.reshape(N, P, G, C // G)
    s1, s2 = h.mean(axis=(1, 3), keepdims=True), (h * xg).mean(axis=(1, 3), keepdims=True)
    dx = (rstd[:, None, :, None] * (h - s1 - xg * s2)).reshape(N, P, C)
    return dx, (dz * xhat).sum(axis=(0, 1)), dz.sum(axis=(0, 1)), dz


# ---------------------------------------------------------------- rotary

def rotary(x, positions, inv_freq, pairs, interleaved, inverse):
    """x [B][T][H][D], positions [B][T][axes]."""
    axis = np.repeat(np.arange(len(pairs)), pairs)
    angle = positions.astype(np.float64)[:, :, axis] * inv_freq.astype(np.float64)
    angle = np.fmod(angle, 2 * math.pi)[:, :, None, :] * (-1 if inverse else 1)
    c, s, R = np.cos(angle), np.sin(angle), len(axis)
    first = np.arange(R) * (2 if interleaved else 1)
    second = first + (1 if interleaved else R)
    y = x.copy()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


# ---------------------------------------------------------------- linear attention

def linear_attention(q, k, v, log_decay, scale, state=None, lengths=None):
    """The recurrence. q [B][T][H][Dk], k, v with as many heads or fewer; state [B][H][Dk][Dv]."""
    B, T, H, Dk = q.shape
    k, v = (np.repeat(a, H // a.shape[2], axis=2) for a in (k, v))
    lam = np.exp(log_decay.astype(np.float64))[:, None, None]
    S = np.zeros((B, H, Dk, v.shape[3])) if state is None else state.astype(np.float64).copy()
    o = np.zeros((B, T, H, v.shape[3]))
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        for t in range(n):
            S[b] = lam * S[b] + k[b, t, :, :, None] * v[b, t, :, None, :]
            o[b, t] = scale * np.einsum("hkv,hk->hv", S[b], q[b, t])
    return o, S


def linear_attention_backward(do, q, k, v, log_decay, scale, state=None, dstate=None, lengths=None):
    """Gradients of q, k, v and the first state, token by token, from the stored states."""
    B, T, H, Dk = q.shape
    Hkv, Dv = k.shape[2], v.shape[3]
    kk, vv = (np.repeat(a, H // Hkv, axis=2) for a in (k, v))
    lam = np.exp(log_decay.astype(np.float64))[:, None, None]
    dq, dk, dv = np.zeros(q.shape), np.zeros(kk.shape), np.zeros(vv.shape)
    first = np.zeros((B, H, Dk, Dv))
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        S = np.zeros((H, Dk, Dv)) if state is None else state[b].astype(np.float64)
        for t in range(n):
            S = lam * S + kk[b, t, :, :, None] * vv[b, t, :, None, :]
            dq[b, t] = scale * np.einsum("hkv,hv->hk", S, do[b, t])
        G = np.zeros((H, Dk, Dv)) if dstate is None else dstate[b].astype(np.float64)
        for t in range(n - 1, -1, -1):
            G = G + scale * q[b, t, :, :, None] * do[b, t, :, None, :]
            dk[b, t] = np.einsum("hkv,hv->hk", G, vv[b, t])
            dv[b, t] = np.einsum("hkv,hk->hv", G, kk[b, t])
            G = lam * G
        first[b] = G
    share = lambda a: a.reshape(B, T, Hkv, H // Hkv, -1).sum(axis=3)  # noqa: E731
    return dq, share(dk), share(dv), first
