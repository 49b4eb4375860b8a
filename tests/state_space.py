"""The operators of a state-space block in 64 bits, with bounds on what fp32 arithmetic may be off."""
import numpy as np

import tokens as K

EPS = K.EPS


def packed(shape):
    return [int(np.prod(shape[i + 1:])) for i in range(len(shape))]


def sigmoid(z):
    return 0.5 * (1 + np.tanh(z / 2))


def silu(z):
    return z * sigmoid(z)


def silu_slope(z):
    s = sigmoid(z)
    return s + z * s * (1 - s)


def close(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its tolerance" % (what, bad.sum(), bad.size,
                                                                           np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)))


# ---------------------------------------------------------------- RMS norm

def rms_norm(h, gamma, eps):
    rstd = 1 / np.sqrt((h ** 2).mean(axis=1, keepdims=True) + eps)
    return h * rstd * gamma, rstd


def rms_norm_backward(dy, h, gamma, rstd, dsum):
    xhat = h * rstd
    g = dy * gamma
    return rstd * (g - xhat * (g * xhat).mean(axis=1, keepdims=True)) + (0 if dsum is None else dsum), (dy * xhat).sum(axis=0)


# ---------------------------------------------------------------- causal convolution

def lengths_of(lengths, B, T):
    return [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]


def causal_conv(x, w, bias, act, state=None, lengths=None):
    """y, the state after, z, and a bound on z's error."""
    B, T, C = x.shape
    taps = w.shape[1]
    y, z, tz = (np.zeros(x.shape) for _ in range(3))
    after = np.zeros((B, taps - 1, C))
    b0 = 0 if bias is None else bias
    for b, n in enumerate(lengths_of(lengths, B, T)):
        rows = np.concatenate((np.zeros((taps - 1, C)) if state is None else state[b], x[b, :n]))
        parts = np.stack([w[:, j] * rows[j:j + n] for j in range(taps)])
        z[b, :n] = parts.sum(axis=0) + b0
        tz[b, :n] = EPS * (taps + 2) * (np.abs(parts).sum(axis=0) + np.abs(b0))
        y[b, :n] = silu(z[b, :n]) if act else z[b, :n]
        after[b] = rows[n:n + taps - 1]
    return y, after, z, tz


def causal_conv_backward(dy, x, w, bias, act, state=None, dstate=None, lengths=None):
    """(dx, dw, dbias, gradient of the state before), and the same of the bounds."""
    B, T, C = x.shape
    taps = w.shape[1]
    _, _, z, tz = causal_conv(x, w, bias, act, state, lengths)
    got = [np.zeros(x.shape), np.zeros(w.shape), np.zeros(C), np.zeros((B, taps - 1, C))]
    tol = [np.zeros(a.shape) for a in got]
    for b, n in enumerate(lengths_of(lengths, B, T)):
        rows = np.concatenate((np.zeros((taps - 1, C)) if state is None else state[b], x[b, :n]))
        dz = dy[b, :n] * (silu_slope(z[b, :n]) if act else 1)
        # no slope's slope is above 0.5; the sigmoid's argument errs by its own last places
        tdz = np.abs(dy[b, :n]) * ((0.5 * tz[b, :n] + (8 + 4 * np.abs(z[b, :n])) * EPS) if act else 0)
        d, t = np.zeros(rows.shape), np.zeros(rows.shape)
        for j in range(taps):
            d[j:j + n] += w[:, j] * dz
            t[j:j + n] += np.abs(w[:, j]) * (tdz + (taps + 2) * EPS * np.abs(dz))
            got[1][:, j] += (dz * rows[j:j + n]).sum(axis=0)
            tol[1][:, j] += ((tdz + 4 * EPS * np.abs(dz)) * np.abs(rows[j:j + n])).sum(axis=0)
        got[2] += dz.sum(axis=0)
        tol[2] += (tdz + 4 * EPS * np.abs(dz)).sum(axis=0)
        if dstate is not None:
            d[n:n + taps - 1] += dstate[b]
            t[n:n + taps - 1] += 2 * EPS * np.abs(dstate[b])
        got[0][b, :n], tol[0][b, :n] = d[taps - 1:], t[taps - 1:]
        got[3][b], tol[3][b] = d[:taps - 1], t[:taps - 1]
    # sums over B*T terms of either sign, in parts: twice the root of their number of last places of the largest sums on the way
    for i in (1, 2):
        tol[i] *= 1 + np.sqrt(B * T) / 2
    return got, tol


# ---------------------------------------------------------------- selective scan

class Scan:
    """One scan in 64 bits with the error that fp32 arithmetic may add up beside every value."""

    def __init__(self, x, delta, A, B, C, D=None, z=None, bias=None, softplus=True, state=None, lengths=None):
        self.x, self.A, self.z = x, A, z
        self.b, self.t, self.d = x.shape
        self.g, self.n = B.shape[2], B.shape[3]
        self.group = np.arange(self.d) // (self.d // self.g)
        self.B, self.C = B, C
        self.D = np.zeros(self.d) if D is None else D
        self.raw = delta + (0 if bias is None else bias)
        self.softplus = softplus
        self.sig = sigmoid(self.raw) if softplus else np.ones(x.shape)
        self.step = np.logaddexp(0, self.raw) if softplus else self.raw
        # the sum's rounding, through the slope of softplus, and a few last places of the result
        self.tstep = EPS * (np.abs(self.raw) * self.sig + (8 if softplus else 0) * np.abs(self.step))
        self.u = self.step * x
        self.tu = np.abs(x) * self.tstep + EPS * np.abs(self.u)
        self.len = lengths_of(lengths, self.b, self.t)
        self.first = np.zeros((self.b, self.d, self.n)) if state is None else state.astype(np.float64)
        self._forward()

    def on(self, t):
        return (np.array(self.len) > t).astype(np.float64)

    def decay(self, t):
        """exp(dt A) of token t and its error; 1 and 0 past the end."""
        e = self.step[:, t, :, None] * self.A
        a = np.exp(e)
        with np.errstate(invalid="ignore"):
            ta = np.where(a > 0, a * (np.abs(self.A) * self.tstep[:, t, :, None] + EPS * (4 * np.abs(e) + 4)), 0.0)
        on = self.on(t)[:, None, None] > 0
        return np.where(on, a, 1.0), np.where(on, ta, 0.0)

    def _forward(self):
        h, th = self.first.copy(), np.zeros(self.first.shape)
        self.h, self.th = [], []
        self.y = np.zeros(self.x.shape)
        self.ty = np.zeros(self.x.shape)
        for t in range(self.t):
            on = self.on(t)[:, None]
            a, ta = self.decay(t)
            B = self.B[:, t][:, self.group] * on[..., None]
            C = self.C[:, t][:, self.group]
            u, tu = self.u[:, t, :, None], self.tu[:, t, :, None]
            th = a * th + ta * np.abs(h) + np.abs(B) * tu + 3 * EPS * (np.abs(a * h) + np.abs(u * B)) * on[..., None]
            h = a * h + u * B
            self.h.append(h)
            self.th.append(th)
            skip = self.D * self.x[:, t]
            self.y[:, t] = on * ((C * h).sum(axis=2) + skip)
            self.ty[:, t] = on * ((np.abs(C) * th).sum(axis=2) + 12 * EPS * ((np.abs(C * h)).sum(axis=2) + np.abs(skip)))
        self.state, self.tstate = h, th
        self.plain, self.tplain = self.y, self.ty
        if self.z is not None:
            there = np.stack([self.on(t) for t in range(self.t)], axis=1)[..., None]
            gate = silu(self.z)
            self.tgate = np.abs(gate) * EPS * (8 + 4 * np.abs(self.z))
            self.ty = there * (self.ty * np.abs(gate) + np.abs(self.y) * (self.tgate + 2 * EPS * np.abs(gate)))
            self.y = there * self.y * gate

    def backward(self, dy, dstate=None):
        """Gradients and their bounds by name."""
        s, got, tol = self, {}, {}
        there = np.stack([s.on(t) for t in range(s.t)], axis=1)[..., None]
        up = dy * there
        if s.z is not None:
            slope = silu_slope(s.z)
            got["dz"] = up * s.plain * slope
            tol["dz"] = np.abs(up) * (s.tplain * np.abs(slope) + np.abs(s.plain) * EPS * (16 + 4 * np.abs(s.z)) * np.maximum(np.abs(slope), 1 - sigmoid(np.abs(s.z))))
            gate = silu(s.z)
            tup = np.abs(up) * (s.tgate + 2 * EPS * np.abs(gate))
            up = up * gate
        else:
            tup = np.zeros(up.shape)
        for f in ("dx", "ddelta"):
            got[f], tol[f] = np.zeros(s.x.shape), np.zeros(s.x.shape)
        for f in ("dB", "dC"):
            got[f], tol[f] = np.zeros(s.B.shape), np.zeros(s.B.shape)
        for f, shape in (("dA", s.A.shape), ("dD", s.d), ("ddelta_bias", s.d)):
            got[f], tol[f] = np.zeros(shape), np.zeros(shape)
        G = np.zeros(s.first.shape) if dstate is None else dstate.astype(np.float64)
        tG = np.zeros(G.shape)
        sizes = {"dA": np.zeros(s.A.shape), "dD": np.zeros(s.d), "ddelta_bias": np.zeros(s.d)}
        per = s.d // s.g
        shared = lambda v: v.reshape(s.b, s.g, per, s.n).sum(axis=2)  # noqa: E731
        for t in range(s.t - 1, -1, -1):
            on = s.on(t)[:, None]
            on3 = on[..., None]
            a, ta = s.decay(t)
            B, C = s.B[:, t][:, s.group] * on3, s.C[:, t][:, s.group] * on3
            g, tg = up[:, t, :, None], tup[:, t, :, None]
            x, u, tu = s.x[:, t], s.u[:, t, :, None], s.tu[:, t, :, None]
            G, tG = G + C * g, tG + np.abs(C) * tg + EPS * (2 * np.abs(C * g) + np.abs(G)) * on3
            before, tbefore = (s.h[t - 1], s.th[t - 1]) if t else (s.first, np.zeros(s.first.shape))
            k = G * a * before * on3
            tk = on3 * (np.abs(a * before) * tG + np.abs(G) * (ta * np.abs(before) + a * tbefore)) + 4 * EPS * np.abs(k)
            du = (G * B).sum(axis=2)
            tdu = (tG * np.abs(B)).sum(axis=2) + 12 * EPS * np.abs(G * B).sum(axis=2)
            live = np.where(np.isfinite(s.A), s.A, 0.0)      # a rate of minus infinity keeps nothing: no gradient comes through it
            got["dx"][:, t] = on * (s.step[:, t] * du) + s.D * up[:, t]
            tol["dx"][:, t] = on * (np.abs(s.step[:, t]) * tdu + s.tstep[:, t] * np.abs(du) + 3 * EPS * np.abs(s.step[:, t] * du)) + \
                np.abs(s.D) * (tup[:, t] + 2 * EPS * np.abs(up[:, t]))
            dstep = x * du * on + (k * live).sum(axis=2)
            tdstep = on * np.abs(x) * (tdu + 2 * EPS * np.abs(du)) + (tk * np.abs(live)).sum(axis=2) + 12 * EPS * np.abs(k * live).sum(axis=2)
            sig = s.sig[:, t]
            got["ddelta"][:, t] = dstep * sig
            tol["ddelta"][:, t] = tdstep * sig + np.abs(dstep) * sig * EPS * (6 + 4 * np.abs(s.raw[:, t]))
            got["ddelta_bias"] += (dstep * sig).sum(axis=0)
            tol["ddelta_bias"] += tol["ddelta"][:, t].sum(axis=0)
            sizes["ddelta_bias"] += np.abs(dstep * sig).sum(axis=0)
            got["dD"] += (up[:, t] * x).sum(axis=0)
            tol["dD"] += (tup[:, t] * np.abs(x)).sum(axis=0)
            sizes["dD"] += np.abs(up[:, t] * x).sum(axis=0)
            st, tst = s.step[:, t, :, None], s.tstep[:, t, :, None]
            got["dA"] += (k * st).sum(axis=0)
            tol["dA"] += (tk * np.abs(st) + np.abs(k) * tst).sum(axis=0)
            sizes["dA"] += np.abs(k * st).sum(axis=0)
            places = EPS * (8 + 2 * np.sqrt(per))
            got["dB"][:, t] = shared(G * u * on3)
            tol["dB"][:, t] = shared(on3 * (tG * np.abs(u) + np.abs(G) * tu + places * np.abs(G * u)))
            got["dC"][:, t] = shared(g * s.h[t] * on3)
            tol["dC"][:, t] = shared(on3 * (tg * np.abs(s.h[t]) + np.abs(g) * s.th[t] + places * np.abs(g * s.h[t])))
            tG = a * tG + ta * np.abs(G) + EPS * np.abs(a * G) * on3
            G = a * G
        for f, size in sizes.items():
            tol[f] += EPS * (8 + 2 * np.sqrt(s.b * s.t)) * size
        got["dstate"], tol["dstate"] = G, tG
        return got, tol
