"""Cases of the operators of a state-space block on tokens: RMS norm with a residual, the same in 8 bits and the product that reads it,
short causal convolutions, selective scans (prompts, single tokens, training).

Fields of every case: op ("norm", "project", "product", "conv", "scan"), dtype ("f32", "bf16", "f16").
norm: rows tokens of c channels; residual (added first, the sum is handed on); train (forward, then backward); gap (elements between the
channels of one token and the next).
project: rows tokens of c channels, normed to 8 bits, times an 8-bit matrix to n channels; residual; bias.
product: m tokens of k channels in 8 bits times an 8-bit matrix to n channels; bias; gap (bytes between rows).
conv: b sequences of t tokens of c channels; taps; act; ragged (sequences of different lengths, padded to t); carry (begins from the inputs
before and hands the last ones on; in training with their gradients); train.
scan: b sequences of t tokens; d channels with n states each; g groups of channels that share B and C; gate; ragged; carry; train.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, **fields):
    return dict({"name": name} if name else {}, **fields)


def _norm(name, rows, c, dtype, residual=True, train=False, gap=0):
    return _case(name, op="norm", rows=rows, c=c, dtype=dtype, residual=residual, train=train, gap=gap)


def _project(name, rows, c, n, dtype, residual=True, bias=False):
    return _case(name, op="project", rows=rows, c=c, n=n, dtype=dtype, residual=residual, bias=bias)


def _product(name, m, n, k, dtype, bias=True, gap=0):
    return _case(name, op="product", m=m, n=n, k=k, dtype=dtype, bias=bias, gap=gap)


def _conv(name, b, t, c, taps, dtype, act="silu", ragged=False, carry=True, train=False):
    return _case(name, op="conv", b=b, t=t, c=c, taps=taps, dtype=dtype, act=act, ragged=ragged, carry=carry, train=train)


def _scan(name, b, t, d, n, dtype, g=1, gate=True, ragged=False, carry=True, train=False):
    return _case(name, op="scan", b=b, t=t, d=d, n=n, dtype=dtype, g=g, gate=gate, ragged=ragged, carry=carry, train=train)


def listed():
    return [
        # A video prompt: 16 frames of 28x28 tokens on their way into a block.
        _norm("norm 12544x2048 bf16", 16 * 28 * 28, 2048, "bf16"),
        # Training on images of an odd size, rows with a gap, single precision.
        _norm("norm train 9800x771 f32", 8 * 35 * 35, 771, "f32", train=True, gap=5),
        # One token of one sequence, latency: normed, then projected.
        _project("project 1x2048x8192 bf16", 1, 2048, 8192, "bf16"),
        # One token of each of 64 sequences that are being answered.
        _project("project 64x4096x8192 f16", 64, 4096, 8192, "f16", bias=True),
        # An image of an odd size to the classes: nothing fits a tile.
        _product("product 1225x1000x771 f32", 35 * 35, 1000, 771, "f32", gap=9),
        # The projection of a video prompt.
        _product("product 12544x8192x4096 bf16", 16 * 28 * 28, 8192, 4096, "bf16", bias=False),
        # One token of each of 64 sequences.
        _conv("conv 1 token b64 bf16", 64, 1, 4096, 4, "bf16"),
        # Training on a batch of images.
        _conv("conv train 3136 b4 bf16", 4, 56 * 56, 2048, 4, "bf16", carry=False, train=True),
        # One token of each of 64 sequences: the states pass through once.
        _scan("scan 1 token b64 bf16", 64, 1, 4096, 16, "bf16"),
        # One video prompt: few channels to fill the chip with.
        _scan("scan 12544 b1 bf16", 1, 16 * 28 * 28, 2048, 16, "bf16"),
        # Prompts of different odd lengths, odd numbers of states and channels, shared by groups, single precision.
        _scan("scan ragged 1225 b8 f32", 8, 35 * 35, 1002, 11, "f32", g=2, ragged=True),
        # Training on a batch of images.
        _scan("scan train 3136 b4 bf16", 4, 56 * 56, 2048, 16, "bf16", carry=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / (400 if case["op"] in ("project", "product") else 10))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "project", "product", "conv", "scan")}
    family = rng.choice(("norm", "project", "product", "conv", "step", "scan", "train"))
    while True:
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        if family == "norm":
            case = _norm(None, _log_int(rng, 1, 32768), _log_int(rng, 16, 8192), dtype, rng.random() < 0.7, rng.random() < 0.5,
                         rng.choice((0, 0, 0, 8, 13)))
        elif family == "project":
            case = _project(None, _log_int(rng, 1, 256), _log_int(rng, 4, 256) * rng.choice((16, 16, 16, 1, 3)),
                            _log_int(rng, 4, 512) * rng.choice((16, 16, 16, 1, 7)), dtype, rng.random() < 0.7, rng.random() < 0.4)
        elif family == "product":
            case = _product(None, _log_int(rng, 1, 16384), _log_int(rng, 4, 512) * rng.choice((16, 16, 16, 1, 7)),
                            _log_int(rng, 4, 512) * rng.choice((16, 16, 16, 1, 3)), dtype, rng.random() < 0.5, rng.choice((0, 0, 16, 5)))
        elif family == "conv":
            t = _log_int(rng, 1, 16384) if rng.random() < 0.7 else 1
            case = _conv(None, _log_int(rng, 1, 64), t, _log_int(rng, 4, 512) * rng.choice((8, 8, 8, 1, 3)), rng.choice((2, 3, 4, 4, 4, 5, 7)),
                         dtype, rng.choice(("silu", "silu", "none")), rng.random() < 0.3, rng.random() < 0.6, rng.random() < 0.4)
        else:
            n = rng.choice((4, 8, 16, 16, 16, 32, 64)) if rng.random() < 0.85 else rng.randrange(1, 65)
            g = rng.choice((1, 1, 1, 2, 4))
            t = _log_int(rng, 1, 4) if family == "step" else _log_int(rng, 16, 16384)
            case = _scan(None, _log_int(rng, 1, 64), t, g * _log_int(rng, 4, 256) * rng.choice((8, 8, 8, 1, 3)), n, dtype, g,
                         rng.random() < 0.7, family != "step" and rng.random() < 0.4, rng.random() < 0.7, family == "train")
        if _cost(case) <= most[case["op"]]:
            return case


# ---------------------------------------------------------------- inputs

def _rand(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _bytes(gen, rows, cols, gap):
    """Rows as they come out of a quantiser: the largest of each is 127 or -127."""
    v = _rand(gen, rows, cols)
    held = torch.zeros((rows, cols + gap), dtype=torch.int8, device="cuda")[:, :cols]
    held.copy_(torch.round(v * (127 / v.abs().amax(dim=1, keepdim=True))))
    return held


def _lengths(case, gen):
    return torch.randint(0, case["t"] + 1, (case["b"],), generator=gen, device="cuda").to(torch.int32) if case["ragged"] else None


def _inputs(case, seed):
    """What the case computes on, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    if case["op"] in ("norm", "project"):
        rows, c = case["rows"], case["c"]
        gap = case.get("gap", 0)
        state = {"x": torch.zeros((rows, c + gap), dtype=dt, device="cuda")[:, :c], "residual": None, "eps": 1e-5,
                 "gamma": 1 + 0.2 * _rand(gen, c)}
        # a residual stream: some channels are many times as large as others
        size = torch.exp(0.7 * _rand(gen, c))
        state["x"].copy_(_rand(gen, rows, c) * size)
        if case["residual"]:
            state["residual"] = (3 * _rand(gen, rows, c) * size).to(dt)
        if case["op"] == "project":
            state["w"] = _bytes(gen, case["n"], c, 0)
            state["w_scale"] = (0.5 + _uniform(gen, case["n"])) * (2.5 / 127 / math.sqrt(c))
            state["bias"] = 0.2 * _rand(gen, case["n"]) if case["bias"] else None
        elif case["train"]:
            state["dy"] = _rand(gen, rows, c).to(dt)
            state["dsum"] = _rand(gen, rows, c).to(dt) if case["residual"] else None
        return state
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"x": _bytes(gen, m, k, case["gap"]), "x_scale": (0.5 + _uniform(gen, m)) * (3.5 / 127),
                "w": _bytes(gen, n, k, case["gap"]), "w_scale": (0.5 + _uniform(gen, n)) * (3.5 / 127 / math.sqrt(k)),
                "bias": 0.2 * _rand(gen, n) if case["bias"] else None}
    b, t = case["b"], case["t"]
    if case["op"] == "conv":
        c, taps = case["c"], case["taps"]
        state = {"x": _rand(gen, b, t, c).to(dt), "w": _rand(gen, c, taps) / math.sqrt(taps), "bias": 0.2 * _rand(gen, c), "state": None,
                 "lengths": _lengths(case, gen)}
        if case["carry"]:
            state["state"] = _rand(gen, b, taps - 1, c).to(dt)
        if case["train"]:
            state["dy"] = _rand(gen, b, t, c).to(dt)
            state["dstate"] = _rand(gen, b, taps - 1, c).to(dt) if case["carry"] else None
        return state
    d, n, g = case["d"], case["n"], case["g"]
    # steps from 0.001 to 0.1 and rates from 1 to n, as such a network begins with: memories from a token to a thousand
    step = torch.exp(math.log(1e-3) + math.log(100.0) * _uniform(gen, d).double())
    state = {"x": _rand(gen, b, t, d).to(dt), "delta": (0.5 * _rand(gen, b, t, d)).to(dt), "delta_bias": torch.log(torch.expm1(step)).float(),
             "A": -(0.7 + 0.6 * _uniform(gen, d, n)) * torch.arange(1, n + 1, device="cuda"),
             "B": _rand(gen, b, t, g, n).to(dt), "C": _rand(gen, b, t, g, n).to(dt), "D": 1 + 0.2 * _rand(gen, d),
             "z": _rand(gen, b, t, d).to(dt) if case["gate"] else None, "state": None, "lengths": _lengths(case, gen)}
    if case["carry"]:
        state["state"] = 0.3 * _rand(gen, b, d, n)
    if case["train"]:
        state["dy"] = _rand(gen, b, t, d).to(dt)
        state["dstate"] = _rand(gen, b, d, n) if case["carry"] else None
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    return state


# ---------------------------------------------------------------- plain forms

def _summed(s):
    return s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)


def _plain_norm(s):
    case, h = s["case"], _summed(s)
    v = h.float()
    rstd = 1 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + s["eps"])
    xhat = v * rstd
    got = {"y": (xhat * s["gamma"]).to(h.dtype)}
    if case["residual"]:
        got["sum"] = h
    if case["train"]:
        dy = s["dy"].float()
        dh = dy * s["gamma"]
        dx = rstd * (dh - xhat * (dh * xhat).mean(dim=1, keepdim=True))
        got["dx"] = (dx if s["dsum"] is None else dx + s["dsum"].float()).to(h.dtype)
        got["dgamma"] = (dy * xhat).sum(dim=0)
    return got


def _scaled(q, scale, w, w_scale, bias, dt):
    # products of whole numbers: exact while their sums stay below 2^24, which those of real inputs do
    y = (q @ w.float().t()) * scale[:, None] * w_scale
    return (y if bias is None else y + bias).to(dt)


def _plain_project(s):
    h = _summed(s)
    v = h.float()
    y = v * (1 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + s["eps"])) * s["gamma"]
    scale = y.abs().amax(dim=1) / 127
    got = {"y": _scaled(torch.round(y / scale[:, None]), scale, s["w"], s["w_scale"], s["bias"], h.dtype), "scale": scale}
    if s["case"]["residual"]:
        got["sum"] = h
    return got


def _plain_product(s):
    return _scaled(s["x"].float(), s["x_scale"], s["w"], s["w_scale"], s["bias"], _TYPES[s["case"]["dtype"]])


def _there(s):
    case = s["case"]
    at = torch.arange(case["t"], device="cuda")
    length = torch.full((case["b"],), case["t"], device="cuda") if s["lengths"] is None else s["lengths"].long()
    return length, (at[None, :] < length[:, None]).float()[:, :, None]


def _silu_slope(z):
    g = 1 / (1 + torch.exp(-z))
    return g * (1 + z * (1 - g))


def _plain_conv(s):
    case, dt = s["case"], s["x"].dtype
    b, t, c, taps = (case[f] for f in ("b", "t", "c", "taps"))
    length, there = _there(s)
    before = torch.zeros((b, taps - 1, c), device="cuda") if s["state"] is None else s["state"].float()
    x = torch.cat((before, s["x"].float() * there), dim=1)
    windows = x.unfold(1, taps, 1)                                             # [b][t][c][taps]
    pre = (windows * s["w"]).sum(dim=3) + s["bias"]
    got = {"y": ((pre / (1 + torch.exp(-pre)) if case["act"] == "silu" else pre) * there).to(dt)}
    last = length[:, None] + torch.arange(taps - 1, device="cuda")             # rows of x that the next call begins from
    pick = last[:, :, None].expand(-1, -1, c)
    if case["carry"]:
        got["state"] = torch.gather(x, 1, pick).to(dt)
    if not case["train"]:
        return got
    dz = s["dy"].float() * there * (_silu_slope(pre) if case["act"] == "silu" else 1)
    got["dw"], got["dbias"] = (dz[..., None] * windows).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    # a row of x is in the windows of the taps tokens from its own on
    dx = (torch.nn.functional.pad(dz, (0, 0, taps - 1, taps - 1)).unfold(1, taps, 1) * s["w"].flip(1)).sum(dim=3)
    if case["carry"]:
        dx = dx.scatter_add(1, pick, s["dstate"].float())
        got["dstate"] = dx[:, :taps - 1].to(dt)
    got["dx"] = (dx[:, taps - 1:] * there).to(dt)
    return got


def _recurrence(a, b):
    """h_t = a_t h_(t-1) + b_t over axis 1, from zero, by doubling."""
    reach, t = 1, a.shape[1]
    while reach < t:
        b = torch.cat((b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]), dim=1)
        a = torch.cat((a[:, :reach], a[:, reach:] * a[:, :-reach]), dim=1)
        reach *= 2
    return b


def _plain_scan(s):
    case, dt = s["case"], s["x"].dtype
    b, t, d, n, g = (case[f] for f in ("b", "t", "d", "n", "g"))
    length, there = _there(s)
    x, raw = s["x"].float() * there, s["delta"].float() + s["delta_bias"]
    step = (torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))) * there
    wide = lambda v: (v.float() * there[..., None]).repeat_interleave(d // g, dim=2)  # noqa: E731
    B, C, A = wide(s["B"]), wide(s["C"]), s["A"]                                         # [b][t][d][n]
    a = torch.exp(step[..., None] * A)
    u = step * x
    enters = u[..., None] * B
    first = torch.zeros((b, d, n), device="cuda") if s["state"] is None else s["state"]
    enters[:, 0] += a[:, 0] * first
    h = _recurrence(a, enters)
    y = (C * h).sum(dim=3) + s["D"] * x
    z = s["z"].float() * there if case["gate"] else None
    gate = z / (1 + torch.exp(-z)) if case["gate"] else 1
    got = {"y": (y * gate).to(dt)}
    if case["carry"]:
        got["state"] = h[:, -1]
    if not case["train"]:
        return got
    up = s["dy"].float() * there
    if case["gate"]:
        got["dz"] = (up * y * _silu_slope(z)).to(dt)
    up = up * gate
    after = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), dim=1)      # what a state is worth to the next token
    enters = up[..., None] * C
    if case["carry"]:
        enters[:, -1] += s["dstate"]
    G = _recurrence(after.flip(1), enters.flip(1)).flip(1)
    kept = torch.cat((first[:, None], h[:, :-1]), dim=1) * a * G         # a_t h_(t-1) dL/dh_t
    du = (G * B).sum(dim=3)
    dstep = (kept * A).sum(dim=3) + x * du
    ddelta = dstep * there / (1 + torch.exp(-raw))
    shared = lambda v: v.view(b, t, g, d // g, n).sum(dim=3).to(dt)  # noqa: E731
    got.update({"dx": ((step * du + s["D"] * up) * there).to(dt), "ddelta": ddelta.to(dt), "ddelta_bias": ddelta.sum(dim=(0, 1)),
                "dA": (kept * step[..., None]).sum(dim=(0, 1)), "dB": shared(G * u[..., None]), "dC": shared(up[..., None] * h),
                "dD": (up * x).sum(dim=(0, 1))})
    if case["carry"]:
        got["dstate"] = G[:, 0] * a[:, 0]
    return got


# ---------------------------------------------------------------- the framework's operators

_handle = None


def _library():
    """One handle per process, as a program keeps it; buffers are the caller's own."""
    global _handle
    if _handle is None:
        import fastconv_amd as F
        _handle = F.load(torch.cuda.current_device(), 1 << 20)
    return _handle


def _workspace(nbytes):
    return torch.empty((nbytes + 3) // 4, dtype=torch.float32, device="cuda") if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    return None if t is None else torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")


def _kept(s):
    """Plan, outputs and workspace of a state, as a program keeps them from call to call."""
    if "plan" in s:
        return s["plan"]
    import fastconv_amd as F
    L, case = _library(), s["case"]
    dtype, dt = {"f32": F.F32, "bf16": F.BF16, "f16": F.F16}[case["dtype"]], _TYPES[case["dtype"]]
    if case["op"] in ("norm", "project"):
        rows, c = case["rows"], case["c"]
        pitch = s["x"].stride(0)
        s["plan"] = plan = L.rms_norm_plan(F.RmsNormShape(rows, c, dtype, s["eps"], pitch, c, c if case["residual"] else pitch, c))
        s["sum"] = torch.empty((rows, c), dtype=dt, device="cuda") if case["residual"] else None
        if case["op"] == "project":
            s["q"] = torch.empty((rows, c), dtype=torch.int8, device="cuda")
            s["scale"] = torch.empty((rows,), device="cuda")
            s["y"] = torch.empty((rows, case["n"]), dtype=dt, device="cuda")
            s["product"] = L.int8_product_plan(F.Int8ProductShape.packed(rows, case["n"], c, dtype))
            s["ws"] = _workspace(s["product"].ws_bytes)
        else:
            s["y"] = torch.empty((rows, c), dtype=dt, device="cuda")
            s["rstd"] = torch.empty((rows,), device="cuda")
            if case["train"]:
                s["dx"], s["dgamma"], s["ws"] = _like(s["x"]), torch.empty_like(s["gamma"]), _workspace(plan.ws_backward_bytes)
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["plan"] = L.int8_product_plan(F.Int8ProductShape(m, n, k, dtype, s["x"].stride(0), s["w"].stride(0), n))
        s["y"], s["ws"] = torch.empty((m, n), dtype=dt, device="cuda"), _workspace(s["plan"].ws_bytes)
    else:
        b, t = case["b"], case["t"]
        if case["op"] == "conv":
            act = F.ACT_SILU if case["act"] == "silu" else F.ACT_NONE
            s["plan"] = L.causal_conv_plan(F.CausalConvShape.packed(b, t, case["c"], case["taps"], dtype, act))
        else:
            s["plan"] = L.selective_scan_plan(F.SelectiveScanShape.packed(b, t, case["d"], case["n"], case["g"], dtype, softplus=True))
        s["y"], s["state_out"] = _like(s["x"]), _like(s["state"])
        if case["train"]:
            for f in ("x", "w", "bias", "state") if case["op"] == "conv" else ("x", "delta", "delta_bias", "A", "B", "C", "D", "z", "state"):
                s["grad_" + f] = _like(s[f])
        s["ws"] = _workspace(max(getattr(s["plan"], "ws_bytes", 0), s["plan"].ws_backward_bytes if case["train"] else 0))
    return s["plan"]


def _own_norm(s):
    L, plan, case = _library(), _kept(s), s["case"]
    x, gamma = s["x"].data_ptr(), s["gamma"].data_ptr()
    L.rms_norm(plan, x, gamma, s["y"].data_ptr(), _ptr(s["residual"]), _ptr(s["sum"]), s["rstd"].data_ptr() if case["train"] else None)
    got = {"y": s["y"]}
    if case["residual"]:
        got["sum"] = s["sum"]
    if case["train"]:
        h = s["sum"].data_ptr() if case["residual"] else x
        L.rms_norm_backward(plan, s["dy"].data_ptr(), h, gamma, s["rstd"].data_ptr(), s["dx"].data_ptr(), s["dgamma"].data_ptr(),
                            _ptr(s["dsum"]), _ptr(s["ws"]))
        got["dx"], got["dgamma"] = s["dx"], s["dgamma"]
    return got


def _own_project(s):
    L, plan, case = _library(), _kept(s), s["case"]
    L.rms_norm_int8(plan, s["x"].data_ptr(), s["gamma"].data_ptr(), s["q"].data_ptr(), s["scale"].data_ptr(), _ptr(s["residual"]),
                    _ptr(s["sum"]))
    L.int8_product(s["product"], s["q"].data_ptr(), s["scale"].data_ptr(), s["w"].data_ptr(), s["w_scale"].data_ptr(), s["y"].data_ptr(),
                   _ptr(s["bias"]), _ptr(s["ws"]))
    return {f: s[f] for f in (("y", "scale", "sum") if case["residual"] else ("y", "scale"))}


def _own_product(s):
    L, plan = _library(), _kept(s)
    L.int8_product(plan, s["x"].data_ptr(), s["x_scale"].data_ptr(), s["w"].data_ptr(), s["w_scale"].data_ptr(), s["y"].data_ptr(),
                   _ptr(s["bias"]), _ptr(s["ws"]))
    return s["y"]


def _own_conv(s):
    L, plan, case = _library(), _kept(s), s["case"]
    x, w, bias, lengths = s["x"].data_ptr(), s["w"].data_ptr(), s["bias"].data_ptr(), _ptr(s["lengths"])
    L.causal_conv(plan, x, w, bias, s["y"].data_ptr(), _ptr(s["state"]), _ptr(s["state_out"]), lengths)
    got = {"y": s["y"]}
    if case["carry"]:
        got["state"] = s["state_out"]
    if case["train"]:
        L.causal_conv_backward(plan, s["dy"].data_ptr(), x, w, bias, s["grad_x"].data_ptr(), s["grad_w"].data_ptr(), s["grad_bias"].data_ptr(),
                               _ptr(s["state"]), _ptr(s["dstate"]), _ptr(s["grad_state"]), lengths, _ptr(s["ws"]))
        got.update({"dx": s["grad_x"], "dw": s["grad_w"], "dbias": s["grad_bias"]})
        if case["carry"]:
            got["dstate"] = s["grad_state"]
    return got


def _own_scan(s):
    L, plan, case = _library(), _kept(s), s["case"]
    given = {f: _ptr(s[f]) for f in ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "lengths")}
    given.update(state_in=_ptr(s["state"]), ws=_ptr(s["ws"]))
    L.selective_scan(plan, y=s["y"].data_ptr(), state_out=_ptr(s["state_out"]), **given)
    got = {"y": s["y"]}
    if case["carry"]:
        got["state"] = s["state_out"]
    if case["train"]:
        names = ["x", "delta", "A", "B", "C", "D", "delta_bias"] + (["z"] if case["gate"] else [])
        L.selective_scan_backward(plan, dy=s["dy"].data_ptr(), dstate_out=_ptr(s["dstate"]), dstate_in=_ptr(s["grad_state"]),
                                  **{"d" + f: _ptr(s["grad_" + f]) for f in names}, **given)
        got.update({"d" + f: s["grad_" + f] for f in names})
        if case["carry"]:
            got["dstate"] = s["grad_state"]
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "project": _own_project, "product": _own_product, "conv": _own_conv, "scan": _own_scan}[op](state)
    return {"norm": _plain_norm, "project": _plain_project, "product": _plain_product, "conv": _plain_conv, "scan": _plain_scan}[op](state)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "norm":
        values = case["rows"] * case["c"]
        moved = (4 if case["residual"] else 2) + ((3 if case["residual"] else 2) if case["train"] else 0)      # dy, dsum, dx
        return {"bytes": float(moved * size * values + 4 * case["c"]), "flops": float((16 if case["train"] else 6) * values)}
    if case["op"] == "project":
        rows, c, n = case["rows"], case["c"], case["n"]
        return {"bytes": float((3 if case["residual"] else 1) * size * rows * c + n * c + size * rows * n + 4 * (rows + c + n)),
                "flops": float(2 * rows * n * c + 10 * rows * c)}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": float(m * k + n * k + size * m * n + 4 * (m + n)), "flops": float(2 * m * n * k)}
    tokens = case["b"] * case["t"]
    if case["op"] == "conv":
        c, taps = case["c"], case["taps"]
        values, carried = tokens * c, (size * case["b"] * (taps - 1) * c * (4 if case["train"] else 2) if case["carry"] else 0)
        return {"bytes": float((4 if case["train"] else 2) * size * values + carried + 4 * c * (taps + 1)),
                "flops": float((6 if case["train"] else 2) * taps * values)}
    d, n, g = case["d"], case["n"], case["g"]
    values, shared = tokens * d, tokens * g * n * 2
    moved = values * (4 if case["gate"] else 3) + shared                # x, delta, z, y; B, C
    if case["train"]:
        moved += values * (4 if case["gate"] else 3) + shared           # dy, dx, ddelta, dz; dB, dC
    carried = 4 * case["b"] * d * n * (4 if case["train"] else 2) if case["carry"] else 0
    return {"bytes": float(size * moved + carried + 4 * d * (n + 2)), "flops": float(values * (n * (30 if case["train"] else 7) + 20))}


# ---------------------------------------------------------------- in 64 bits

def _exact_rows(case, s):
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
    got = {"sum": h} if case["residual"] else {}
    h = h.to(s["x"].dtype).double()
    return h, torch.rsqrt(h.square().mean(dim=1, keepdim=True) + s["eps"]), got


def _exact_norm(case, s):
    h, rstd, got = _exact_rows(case, s)
    gamma = s["gamma"].double()
    got["y"] = h * rstd * gamma
    if case["train"]:
        dy = s["dy"].double()
        got["dgamma"] = torch.mv((h * dy).t(), rstd[:, 0])
        along = (dy * gamma * h).sum(dim=1, keepdim=True) * rstd.pow(3) / case["c"]
        got["dx"] = dy * gamma * rstd - h * along + (0 if s["dsum"] is None else s["dsum"].double())
    return got


def _exact_project(case, s):
    h, rstd, got = _exact_rows(case, s)
    y = h * s["gamma"].double() * rstd
    top = y.abs().max(dim=1, keepdim=True).values
    q = torch.round(y * 127 / top)
    got["scale"] = top[:, 0] / 127
    got["y"] = torch.mm(q, s["w"].double().t()) * (top / 127) * s["w_scale"].double() + (0 if s["bias"] is None else s["bias"].double())
    return got


def _exact_product(case, s):
    if case["m"] * case["n"] * case["k"] > 1e13:
        return None
    y = torch.mm(s["x"].double(), s["w"].double().t())
    y = y * s["x_scale"].double()[:, None] * s["w_scale"].double()
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_conv(case, s):
    b, t, c, taps = (case[f] for f in ("b", "t", "c", "taps"))
    length = [t] * b if s["lengths"] is None else s["lengths"].tolist()
    w, bias = s["w"].double(), s["bias"].double()
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    got = {"y": zeros(b, t, c)}
    if case["carry"]:
        got["state"] = zeros(b, taps - 1, c)
    if case["train"]:
        got.update({"dx": zeros(b, t, c), "dw": zeros(c, taps), "dbias": zeros(c)})
        if case["carry"]:
            got["dstate"] = zeros(b, taps - 1, c)
    for i, m in enumerate(length):
        x = zeros(taps - 1 + m, c)
        if s["state"] is not None:
            x[:taps - 1] = s["state"][i].double()
        x[taps - 1:] = s["x"][i, :m].double()
        pre = bias.expand(m, c).clone()
        for j in range(taps):
            pre += w[:, j] * x[j:j + m]
        sig = torch.sigmoid(pre)
        got["y"][i, :m] = pre * sig if case["act"] == "silu" else pre
        if case["carry"]:
            got["state"][i] = x[m:m + taps - 1]
        if case["train"]:
            dz = s["dy"][i, :m].double() * (sig + pre * sig * (1 - sig) if case["act"] == "silu" else 1)
            got["dbias"] += dz.sum(dim=0)
            dx = torch.zeros_like(x)
            for j in range(taps):
                got["dw"][:, j] += (dz * x[j:j + m]).sum(dim=0)
                dx[j:j + m] += w[:, j] * dz
            if case["carry"]:
                dx[m:m + taps - 1] += s["dstate"][i].double()
                got["dstate"][i] = dx[:taps - 1]
            got["dx"][i, :m] = dx[taps - 1:]
    return got


def _exact_scan(case, s):
    b, t, d, n, g = (case[f] for f in ("b", "t", "d", "n", "g"))
    size = b * d * n
    if t * (3 if case["train"] else 1) * max(2e-4, size * 4e-11) > 12 or (case["train"] and t * size * 8 > 60e9):
        return None
    A, skip = s["A"].double(), s["D"].double()
    length = torch.tensor([t] * b if s["lengths"] is None else s["lengths"].tolist(), device="cuda").view(b, 1)
    h = torch.zeros((b, d, n), dtype=torch.float64, device="cuda") if s["state"] is None else s["state"].double()
    first = h
    group = torch.arange(d, device="cuda") // (d // g)

    def token(i):
        raw = s["delta"][:, i].double() + s["delta_bias"].double()
        return i < length, torch.logaddexp(raw, torch.zeros_like(raw)), raw, s["x"][:, i].double(), s["B"][:, i].double()[:, group], s["C"][:, i].double()[:, group]

    y = torch.zeros((b, t, d), dtype=torch.float64, device="cuda")
    states = []
    for i in range(t):      # the recurrence, a token at a time
        on, step, _, x, B, C = token(i)
        h = torch.where(on[..., None], torch.exp(step[..., None] * A) * h + (step * x)[..., None] * B, h)
        y[:, i] = ((C * h).sum(dim=2) + skip * x) * on
        if case["train"]:
            states.append(h)
    plain = y
    if case["gate"]:
        z = s["z"].double()
        y = y * z * torch.sigmoid(z)
    got = {"y": y}
    if case["carry"]:
        got["state"] = h
    if not case["train"]:
        return got
    up = s["dy"].double()
    if case["gate"]:
        sig = torch.sigmoid(z)
        got["dz"] = up * plain * (sig + z * sig * (1 - sig))
        up = up * z * sig
    for f in ("x", "delta"):
        got["d" + f] = torch.zeros((b, t, d), dtype=torch.float64, device="cuda")
    for f in ("B", "C"):
        got["d" + f] = torch.zeros((b, t, g, n), dtype=torch.float64, device="cuda")
    got.update({"dA": torch.zeros_like(A), "dD": torch.zeros_like(skip), "ddelta_bias": torch.zeros_like(skip)})
    G = torch.zeros((b, d, n), dtype=torch.float64, device="cuda") if s["dstate"] is None else s["dstate"].double()
    for i in range(t - 1, -1, -1):      # G: of the state after token i
        on, step, raw, x, B, C = token(i)
        here = up[:, i] * on
        G = G + here[..., None] * C
        live = G * on[..., None]
        a = torch.exp(step[..., None] * A)
        through = live * a * (states[i - 1] if i else first)
        du = (live * B).sum(dim=2)
        got["dx"][:, i] = step * du + skip * here
        ddelta = ((through * A).sum(dim=2) + x * du) * torch.sigmoid(raw)
        got["ddelta"][:, i] = ddelta
        got["ddelta_bias"] += ddelta.sum(dim=0)
        got["dD"] += (here * x).sum(dim=0)
        got["dA"] += (through * step[..., None]).sum(dim=0)
        got["dB"][:, i] = (live * (step * x)[..., None]).view(b, g, d // g, n).sum(dim=2)
        got["dC"][:, i] = (here[..., None] * states[i]).view(b, g, d // g, n).sum(dim=2)
        G = torch.where(on[..., None], a * G, G)
    if case["carry"]:
        got["dstate"] = G
    return got


def exact(case, seed):
    s = _inputs(case, seed)
    return {"norm": _exact_norm, "project": _exact_project, "product": _exact_product, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](case, s)
