"""Cases of the token operators: group norm with an activation over channels-last pixels, rotary positions with several
axes, linear attention with a decay for each head (prompts, single tokens, training).

Fields of every case: op ("norm", "rotary", "attention"), dtype ("f32", "bf16", "f16").
norm: n images of p pixels with c channels in g groups; act; train (forward, then backward); gap (elements between the
channels of one pixel and the next).
rotary: b sequences over a grid of frames x rows x cols tokens; hq query and hk key heads of d channels; s0, s1, s2 (pairs
rotated by the time, the row and the column; the other channels pass); interleaved (pairs of neighbours, not of halves);
inverse (the backward pass).
attention: b sequences of t tokens; h heads, hkv key/value heads; dk, dv; ragged (sequences of different lengths, padded
to t); carry (begins from a state and hands one on; in training with its gradient); train (forward, then backward).
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _norm(name, n, p, c, g, dtype, act="silu", train=False, gap=0):
    return _named(name, {"op": "norm", "n": n, "p": p, "c": c, "g": g, "dtype": dtype, "act": act, "train": train, "gap": gap})


def _rotary(name, b, frames, rows, cols, hq, hk, d, sections, dtype, interleaved=False, inverse=False):
    return _named(name, {"op": "rotary", "b": b, "frames": frames, "rows": rows, "cols": cols, "hq": hq, "hk": hk, "d": d,
                         "s0": sections[0], "s1": sections[1], "s2": sections[2], "dtype": dtype, "interleaved": interleaved,
                         "inverse": inverse})


def _attention(name, b, t, h, hkv, dk, dv, dtype, ragged=False, carry=True, train=False):
    return _named(name, {"op": "attention", "b": b, "t": t, "h": h, "hkv": hkv, "dk": dk, "dv": dv, "dtype": dtype,
                         "ragged": ragged, "carry": carry, "train": train})


def _named(name, case):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One image, latency: the deep layers of a trunk.
        _norm("norm 512@14 n1 bf16", 1, 14 * 14, 512, 32, "bf16"),
        # A size off every grid: groups of six channels, pixels with a gap between them.
        _norm("norm 192@35 n8 f16", 8, 35 * 35, 192, 32, "f16", act="gelu", gap=24),
        # Large images on a batch, few channels: two channels a group.
        _norm("norm 64@224 n32 bf16", 32, 224 * 224, 64, 32, "bf16"),
        # Training on a batch: forward and backward in single precision.
        _norm("norm train 256@56 n32 f32", 32, 56 * 56, 256, 32, "f32", train=True),
        # One token of each of 32 sequences that are being answered.
        _rotary("rotary 1 token b32 bf16", 32, 1, 1, 1, 32, 8, 128, (16, 24, 24), "bf16"),
        # A video prompt: 16 frames of 28x28 tokens, shared key heads.
        _rotary("rotary 16x28x28 b2 bf16", 2, 16, 28, 28, 32, 8, 128, (16, 24, 24), "bf16"),
        # Gradient over images of an odd size; 64 of 80 channels rotated, pairs of neighbours.
        _rotary("rotary grad 35x35 b8 f32", 8, 1, 35, 35, 12, 12, 80, (0, 16, 16), "f32", interleaved=True, inverse=True),
        # One token of one sequence, latency.
        _attention("attn 1 token b1 bf16", 1, 1, 16, 16, 128, 128, "bf16"),
        # One token of each of 64 sequences: the states pass through once.
        _attention("attn 1 token b64 f16", 64, 1, 16, 16, 128, 128, "f16"),
        # One video prompt: 16 frames of 28x28 tokens, few rows to fill the chip with.
        _attention("attn 12544 b1 bf16", 1, 16 * 28 * 28, 16, 16, 128, 128, "bf16"),
        # Prompts of different odd lengths with shared key/value heads and other value sizes, single precision.
        _attention("attn ragged 1225 b8 f32", 8, 35 * 35, 12, 4, 64, 96, "f32", ragged=True),
        # Training on a batch of images.
        _attention("attn train 3136 b8 bf16", 8, 56 * 56, 16, 16, 64, 64, "bf16", carry=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    family = rng.choice(("norm", "norm", "rotary", "prompt", "train", "step"))
    while True:
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        if family == "norm":
            g = rng.choice((1, 8, 16, 32, 32))
            c = g * _log_int(rng, 1, 1024 // g)
            train = rng.random() < 0.4      # a slope that jumps has no gradient to compare at the jump
            case = _norm(None, _log_int(rng, 1, 64), _log_int(rng, 1, 224 * 224), c, g, dtype,
                         rng.choice(("silu", "silu", "gelu", "none" if train else "relu", "none")), train,
                         rng.choice((0, 0, 0, 8, 13)))
            if case["p"] * c < 16 * g:      # a group of a few values is its own statistics
                continue
        elif family == "rotary":
            d = rng.choice((32, 64, 80, 96, 128, 128, 256))
            pairs = d // 2 if rng.random() < 0.6 else rng.randrange(3, d // 2 + 1)
            one = rng.randrange(0, pairs // 2 + 1)
            two = (pairs - one) // 2
            hk = rng.choice((1, 2, 4, 8, 12))
            frames, rows, cols = rng.choice(((1, 1, 1), (1, 0, 0), (1, 0, 0), (_log_int(rng, 1, 64), 0, 0)))
            case = _rotary(None, _log_int(rng, 1, 64), frames, rows or _log_int(rng, 2, 64), cols or _log_int(rng, 2, 64),
                           hk * rng.choice((1, 2, 4)), hk, d, (one, two, pairs - one - two), dtype, rng.random() < 0.4,
                           rng.random() < 0.4)
        else:
            hkv, same = rng.choice((1, 2, 4, 8, 16)), rng.random() < 0.7
            dk = rng.choice((16, 32, 64, 64, 128, 128)) if rng.random() < 0.85 else rng.randrange(8, 129)
            dv = dk if same else rng.choice((16, 40, 64, 96, 128, 200, 256))
            t = _log_int(rng, 1, 16) if family == "step" else _log_int(rng, 16, 16384)
            case = _attention(None, _log_int(rng, 1, 64), t, hkv * rng.choice((1, 1, 2, 4)), hkv, dk, dv, dtype,
                              family != "step" and rng.random() < 0.4, rng.random() < 0.7, family == "train")
        if _cost(case) <= most:
            return case


# ---------------------------------------------------------------- inputs

def _rand(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _inputs(case, seed):
    """What the case computes on, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    if case["op"] == "norm":
        n, p, c = case["n"], case["p"], case["c"]
        # features with a mean and a scale of their own in each channel, as a convolution leaves them
        x = torch.empty((n, p, c + case["gap"]), dtype=dt, device="cuda")[:, :, :c]
        x.copy_(_rand(gen, n, p, c) * (0.5 + torch.rand((c,), generator=gen, device="cuda")) + 0.5 * _rand(gen, c))
        state = {"x": x, "gamma": 1 + 0.2 * _rand(gen, c), "beta": 0.2 * _rand(gen, c), "eps": 1e-5}
        if case["train"]:
            state["dy"] = _rand(gen, n, p, c).to(dt)
        return state
    if case["op"] == "rotary":
        b, t = case["b"], case["frames"] * case["rows"] * case["cols"]
        # the grid of each sequence begins at a place of its own; times run longer where the type is coarse anyway
        first = torch.randint(0, 128 if case["dtype"] == "f32" else 4096, (b, 1), generator=gen, device="cuda")
        at = torch.arange(t, device="cuda")
        grid = case["rows"] * case["cols"]
        positions = torch.stack((first + at // grid, (first % 64) + at % grid // case["cols"],
                                 (first % 32) + at % case["cols"]), dim=-1).to(torch.int32).contiguous()
        ladders = [10000.0 ** (-torch.arange(s, device="cuda", dtype=torch.float64) / max(s, 1))
                   for s in (case["s0"], case["s1"], case["s2"])]
        return {"q": _rand(gen, b, t, case["hq"], case["d"]).to(dt), "k": _rand(gen, b, t, case["hk"], case["d"]).to(dt),
                "positions": positions, "inv_freq": torch.cat(ladders).float()}
    b, t, h, hkv, dk, dv = (case[f] for f in ("b", "t", "h", "hkv", "dk", "dv"))
    state = {"q": _rand(gen, b, t, h, dk).to(dt), "k": _rand(gen, b, t, hkv, dk).to(dt), "v": _rand(gen, b, t, hkv, dv).to(dt),
             # half-lives from a few tokens to a few thousand
             "log_decay": -torch.exp2(-1.0 - 10.0 * torch.rand((h,), generator=gen, device="cuda")),
             "scale": dk ** -0.5, "lengths": None, "state": None}
    if case["ragged"]:
        state["lengths"] = torch.randint(0, t + 1, (b,), generator=gen, device="cuda").to(torch.int32)
    if case["carry"]:
        state["state"] = _rand(gen, b, h, dk, dv)
    if case["train"]:
        state["do"] = _rand(gen, b, t, h, dv).to(dt)
        state["dstate"] = _rand(gen, b, h, dk, dv) if case["carry"] else None
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    return state


# ---------------------------------------------------------------- plain forms

def _activation(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _activation_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _plain_norm(s):
    case = s["case"]
    n, p, c, g = case["n"], case["p"], case["c"], case["g"]
    x = s["x"].float().reshape(n, p, g, c // g)
    gamma, beta = s["gamma"].view(g, c // g), s["beta"].view(g, c // g)
    xhat = x - x.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((xhat * xhat).mean(dim=(1, 3), keepdim=True) + s["eps"])
    xhat = xhat * rstd
    z = xhat * gamma + beta
    y = _activation(z, case["act"]).reshape(n, p, c).to(s["x"].dtype)
    if not case["train"]:
        return y
    dz = s["dy"].float().view(n, p, g, c // g) * _activation_slope(z, case["act"])
    dgamma, dbeta = (dz * xhat).sum(dim=(0, 1)).reshape(c), dz.sum(dim=(0, 1)).reshape(c)
    dz = dz * gamma
    dx = rstd * (dz - dz.mean(dim=(1, 3), keepdim=True) - xhat * (dz * xhat).mean(dim=(1, 3), keepdim=True))
    return {"y": y, "dx": dx.reshape(n, p, c).to(s["x"].dtype), "dgamma": dgamma, "dbeta": dbeta}


def _turn(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    v = x.float()
    a, b = (v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]) if interleaved else (v[..., :pairs], v[..., pairs:2 * pairs])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, v[..., 2 * pairs:]), dim=-1).to(x.dtype)


def _plain_rotary(s):
    case, at = s["case"], s["positions"].float()
    of_axis = torch.cat((at[..., 0:1].expand(-1, -1, case["s0"]), at[..., 1:2].expand(-1, -1, case["s1"]),
                         at[..., 2:3].expand(-1, -1, case["s2"])), dim=-1)
    angle = (of_axis * s["inv_freq"])[:, :, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)
    sin = -sin if case["inverse"] else sin
    return {"q": _turn(s["q"], cos, sin, case["interleaved"]), "k": _turn(s["k"], cos, sin, case["interleaved"])}


def _chunked(q, k, v, log_decay, state):
    """sum over j <= i of decay^(i - j) (q_i . k_j) v_j + decay^(i + 1) state^T q_i, heads before tokens, in chunks."""
    b, h, t, _ = q.shape
    c = min(t, 128)
    pad, n = -t % c, -(-t // c)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)).view(b, h, n, c, x.shape[-1]) for x in (q, k, v))
    g = log_decay.view(h, 1, 1)
    i = torch.arange(c, device=q.device, dtype=torch.float32)
    gap = i[:, None] - i[None, :]
    near = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0)
    out = ((q @ k.transpose(-1, -2)) * near[:, None]) @ v
    part = (k * torch.exp(g * (c - 1 - i)).view(h, 1, c, 1)).transpose(-1, -2) @ v
    m = torch.arange(n, device=q.device, dtype=torch.float32)
    gap = m[:, None] - 1 - m[None, :]
    far = torch.where(gap >= 0, torch.exp(g * c * gap.clamp(min=0)), 0.0)
    enters = (far @ part.reshape(b, h, n, -1)).view_as(part)
    if state is not None:
        enters = enters + torch.exp(g * c * m.view(1, n, 1)).view(h, n, 1, 1) * state[:, :, None]
    out = out + (q * torch.exp(g * (i + 1)).view(h, 1, c, 1)) @ enters
    return out.reshape(b, h, n * c, -1)[:, :, :t]


def _plain_attention(s):
    case, scale, g, dt = s["case"], s["scale"], s["log_decay"], s["q"].dtype
    b, t, h, hkv = case["b"], case["t"], case["h"], case["hkv"]
    at = torch.arange(t, device="cuda")
    length = torch.full((b,), t, device="cuda") if s["lengths"] is None else s["lengths"].long()
    there = (at[None, :] < length[:, None]).float().view(b, 1, t, 1)
    q = s["q"].float().transpose(1, 2) * there
    k, v = (x.float().transpose(1, 2).repeat_interleave(h // hkv, dim=1) * there for x in (s["k"], s["v"]))
    # what a token is worth at the end of its sequence
    left = (length[:, None] - 1 - at[None, :]).clamp(min=0).float()
    left = torch.exp(g.view(1, h, 1) * left[:, None, :])[..., None] * there
    whole = torch.exp(g.view(1, h) * length.float()[:, None]).view(b, h, 1, 1)
    got = {"o": (_chunked(q, k, v, g, s["state"]) * scale * there).transpose(1, 2).contiguous().to(dt)}
    if case["carry"]:
        got["state"] = (k * left).transpose(-1, -2) @ v + whole * s["state"]
    if not case["train"]:
        return got
    do = s["do"].float().transpose(1, 2) * there * scale
    initial = None if s["state"] is None else s["state"].transpose(-1, -2)
    dq = _chunked(do, v, k, g, initial)
    dk = _chunked(v.flip(2), do.flip(2), q.flip(2), g, None).flip(2)
    dv = _chunked(k.flip(2), q.flip(2), do.flip(2), g, None).flip(2)
    if case["carry"]:
        dk = dk + left * (v @ s["dstate"].transpose(-1, -2))
        dv = dv + left * (k @ s["dstate"])
        since = torch.exp(g.view(1, h, 1) * (at + 1).float()).view(1, h, t, 1)
        got["dstate"] = (q * since).transpose(-1, -2) @ do + whole * s["dstate"]
    shared = lambda x: (x * there).view(b, hkv, h // hkv, t, -1).sum(dim=2)  # noqa: E731
    got["dq"] = (dq * there).transpose(1, 2).contiguous().to(dt)
    got["dk"] = shared(dk).transpose(1, 2).contiguous().to(dt)
    got["dv"] = shared(dv).transpose(1, 2).contiguous().to(dt)
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


def _kept(s):
    """Plan, outputs and workspace of a state, as a program keeps them from call to call."""
    if "plan" in s:
        return s["plan"]
    import fastconv_amd as F
    L, case = _library(), s["case"]
    dtype = {"f32": F.F32, "bf16": F.BF16, "f16": F.F16}[case["dtype"]]
    if case["op"] == "norm":
        act = {"none": F.ACT_NONE, "relu": F.ACT_RELU, "silu": F.ACT_SILU, "gelu": F.ACT_GELU}[case["act"]]
        n, p, c = case["n"], case["p"], case["c"]
        s["plan"] = L.group_norm_plan(F.GroupNormShape(n, p, c, case["g"], dtype, act, s["eps"], s["x"].stride(0), s["x"].stride(1),
                                                       p * c, c))
        s["y"] = torch.empty((n, p, c), dtype=s["x"].dtype, device="cuda")
        s["mean"], s["rstd"] = (torch.empty((n, case["g"]), device="cuda") for _ in range(2))
        if case["train"]:
            s["dx"] = torch.empty_strided(s["x"].shape, s["x"].stride(), dtype=s["x"].dtype, device="cuda")
            s["dgamma"], s["dbeta"] = torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
        s["ws"] = _workspace(max(s["plan"].ws_bytes, s["plan"].ws_backward_bytes if case["train"] else 0))
    elif case["op"] == "rotary":
        s["plan"] = F.RotaryShape.packed(case["b"], s["q"].shape[1], case["hq"], case["hk"], case["d"],
                                         (case["s0"], case["s1"], case["s2"]), dtype, case["interleaved"])
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    else:
        s["plan"] = L.linear_attention_plan(F.LinearAttentionShape.packed(
            case["b"], case["t"], case["h"], case["hkv"], case["dk"], case["dv"], dtype, s["scale"]))
        s["o"] = torch.empty((case["b"], case["t"], case["h"], case["dv"]), dtype=s["q"].dtype, device="cuda")
        s["state_out"] = torch.empty_like(s["state"]) if case["carry"] else None
        if case["train"]:
            s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[x]) for x in ("q", "k", "v"))
            s["dstate_in"] = torch.empty_like(s["state"]) if case["carry"] else None
        s["ws"] = _workspace(max(s["plan"].ws_bytes, s["plan"].ws_backward_bytes if case["train"] else 0))
    return s["plan"]


def _own_norm(s):
    L, plan, train = _library(), _kept(s), s["case"]["train"]
    mean, rstd = (s["mean"].data_ptr(), s["rstd"].data_ptr()) if train else (None, None)
    L.group_norm(plan, s["x"].data_ptr(), s["gamma"].data_ptr(), s["beta"].data_ptr(), s["y"].data_ptr(), mean, rstd, _ptr(s["ws"]))
    if not train:
        return s["y"]
    L.group_norm_backward(plan, s["dy"].data_ptr(), s["x"].data_ptr(), s["gamma"].data_ptr(), s["beta"].data_ptr(), mean, rstd,
                          s["dx"].data_ptr(), s["dgamma"].data_ptr(), s["dbeta"].data_ptr(), _ptr(s["ws"]))
    return {f: s[f] for f in ("y", "dx", "dgamma", "dbeta")}


def _own_rotary(s):
    shape = _kept(s)
    _library().rotary(shape, s["q"].data_ptr(), s["k"].data_ptr(), s["positions"].data_ptr(), s["inv_freq"].data_ptr(),
                      s["q_out"].data_ptr(), s["k_out"].data_ptr(), s["case"]["inverse"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_attention(s):
    L, plan, case = _library(), _kept(s), s["case"]
    q, k, v, g = s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["log_decay"].data_ptr()
    L.linear_attention(plan, q, k, v, g, s["o"].data_ptr(), _ptr(s["state"]), _ptr(s["state_out"]), _ptr(s["lengths"]), _ptr(s["ws"]))
    got = {"o": s["o"]}
    if case["carry"]:
        got["state"] = s["state_out"]
    if case["train"]:
        L.linear_attention_backward(plan, s["do"].data_ptr(), q, k, v, g, s["dq"].data_ptr(), s["dk"].data_ptr(), s["dv"].data_ptr(),
                                    _ptr(s["state"]), _ptr(s["dstate"]), _ptr(s["dstate_in"]), _ptr(s["lengths"]), _ptr(s["ws"]))
        got.update({f: s[f] for f in ("dq", "dk", "dv")})
        if case["carry"]:
            got["dstate"] = s["dstate_in"]
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_norm if op == "norm" else _own_rotary if op == "rotary" else _own_attention)(state)
    return (_plain_norm if op == "norm" else _plain_rotary if op == "rotary" else _plain_attention)(state)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "norm":
        values = case["n"] * case["p"] * case["c"]
        moved, ops = (5, 60) if case["train"] else (2, 20)      # x, y; then x, dy, dx
        return {"bytes": float(moved * size * values + 16 * case["c"]), "flops": float(ops * values)}
    if case["op"] == "rotary":
        tokens = case["b"] * case["frames"] * case["rows"] * case["cols"]
        pairs = case["s0"] + case["s1"] + case["s2"]
        return {"bytes": float(2 * size * tokens * (case["hq"] + case["hk"]) * case["d"] + 12 * tokens + 4 * pairs),
                "flops": float(6 * tokens * (case["hq"] + case["hk"]) * pairs)}
    tokens, h, hkv, dk, dv = case["b"] * case["t"], case["h"], case["hkv"], case["dk"], case["dv"]
    inputs, state = tokens * (h * dk + hkv * (dk + dv)), 4 * case["b"] * h * dk * dv
    nbytes, nflops = size * (inputs + tokens * h * dv), 4 * dk * dv     # the state takes a token in, and answers for it
    if case["train"]:
        nbytes, nflops = nbytes + size * (2 * inputs + tokens * h * dv), 14 * dk * dv      # q, k, v, do in, dq, dk, dv out
    if case["carry"]:
        nbytes += state * (5 if case["train"] else 2)
    return {"bytes": float(nbytes + 4 * h), "flops": float(nflops * tokens * h)}


# ---------------------------------------------------------------- in 64 bits

def _exact_norm(case, s):
    n, c, g = case["n"], case["c"], case["g"]
    wide = lambda v: v.double().repeat_interleave(c // g)  # noqa: E731
    gamma, beta = s["gamma"].double(), s["beta"].double()
    got = {f: [] for f in ("y", "dx", "dgamma", "dbeta")}
    for image in range(n):
        x = s["x"][image].double()
        by_group = x.t().reshape(g, -1)      # a group's channels, each with all its pixels
        mean, var = by_group.mean(dim=1), by_group.var(dim=1, unbiased=False)
        rstd = (var + s["eps"]).rsqrt()
        xhat = (x - wide(mean)) * wide(rstd)
        z = xhat * gamma + beta
        normal = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        y = {"none": z, "relu": z.relu(), "silu": z * torch.sigmoid(z), "gelu": z * normal}[case["act"]]
        got["y"].append(y.to(torch.float64))
        if case["train"]:
            sig = torch.sigmoid(z)
            slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": sig + z * sig * (1 - sig),
                     "gelu": normal + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)}[case["act"]]
            dz = s["dy"][image].double() * slope
            got["dgamma"].append((dz * xhat).sum(dim=0))
            got["dbeta"].append(dz.sum(dim=0))
            dh = dz * gamma
            m = case["p"] * (c // g)
            first, second = dh.t().reshape(g, -1).sum(dim=1) / m, (dh * xhat).t().reshape(g, -1).sum(dim=1) / m
            got["dx"].append((dh - wide(first) - xhat * wide(second)) * wide(rstd))
    if not case["train"]:
        return torch.stack(got["y"])
    return {"y": torch.stack(got["y"]), "dx": torch.stack(got["dx"]), "dgamma": torch.stack(got["dgamma"]).sum(dim=0),
            "dbeta": torch.stack(got["dbeta"]).sum(dim=0)}


def _exact_rotary(case, s):
    axis = torch.tensor([0] * case["s0"] + [1] * case["s1"] + [2] * case["s2"], device="cuda")
    angle = s["positions"].double()[:, :, axis] * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)[:, :, None, :]
    pairs, got = axis.numel(), {}
    for name in ("q", "k"):
        x = s[name].double()
        y = x.clone()
        first = torch.arange(pairs, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else pairs)
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        got[name] = y
    return got


def _exact_attention(case, s):
    b, t, h, hkv, dk, dv = (case[f] for f in ("b", "t", "h", "hkv", "dk", "dv"))
    rounds = (3 if case["train"] else 1) * t
    if rounds * max(1e-4, b * h * dk * dv * 1.5e-11) > 12:
        return None
    group = h // hkv
    q, k, v = s["q"].double(), s["k"].double().repeat_interleave(group, dim=2), s["v"].double().repeat_interleave(group, dim=2)
    decay = torch.exp(s["log_decay"].double()).view(1, h, 1, 1)
    length = [t] * b if s["lengths"] is None else s["lengths"].tolist()
    length = torch.tensor(length, device="cuda").view(b, 1, 1, 1)
    scale = s["scale"]
    S = torch.zeros((b, h, dk, dv), dtype=torch.float64, device="cuda") if s["state"] is None else s["state"].double()
    o = torch.zeros((b, t, h, dv), dtype=torch.float64, device="cuda")
    dq, dkk, dvv = (torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda") if case["train"] else None for d in (dk, dk, dv))
    do = s["do"].double() if case["train"] else None
    for i in range(t):      # the recurrence, a token at a time
        on = i < length
        S = torch.where(on, decay * S + k[:, i, :, :, None] * v[:, i, :, None, :], S)
        o[:, i] = (scale * on * S * q[:, i, :, :, None]).sum(dim=2)
        if case["train"]:
            dq[:, i] = (scale * on * S * do[:, i, :, None, :]).sum(dim=3)
    got = {"o": o}
    if case["carry"]:
        got["state"] = S
    if case["train"]:
        dS = torch.zeros_like(S) if s["dstate"] is None else s["dstate"].double()
        for i in range(t - 1, -1, -1):      # dS: of the state after token i
            on = i < length
            dS = torch.where(on, dS + scale * q[:, i, :, :, None] * do[:, i, :, None, :], dS)
            dkk[:, i] = (on * dS * v[:, i, :, None, :]).sum(dim=3)
            dvv[:, i] = (on * dS * k[:, i, :, :, None]).sum(dim=2)
            dS = torch.where(on, decay * dS, dS)
        if case["carry"]:
            got["dstate"] = dS
        got["dq"] = dq
        got["dk"] = dkk.view(b, t, hkv, group, dk).sum(dim=3)
        got["dv"] = dvv.view(b, t, hkv, group, dv).sum(dim=3)
    return got


def exact(case, seed):
    s = _inputs(case, seed)
    return (_exact_norm if case["op"] == "norm" else _exact_rotary if case["op"] == "rotary" else _exact_attention)(case, s)
