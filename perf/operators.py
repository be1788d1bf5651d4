"""Cases of the sequence operators (pnp_amd.seqops): the residual's addition with the RMS norm, the
product in 8-bit integers, the short causal convolution and the selective state space scan.

``run`` computes an operator in its plain form (elementary torch operations, fp32 inside, rounded once),
or, where ``own`` is true, by the framework's entry points.  ``exact`` is the operator's definition in
fp64, its gradients by differentiation of that definition."""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # the residual stream of the learner's replay windows: batch 512, 32 steps and the next one
        {"name": "norm windows f32", "op": "norm", "rows": 512 * 33, "dim": 256, "type": "f32", "residual": True},
        # a long batch of wide rows, training in 16 bits
        {"name": "norm wide bf16", "op": "norm", "rows": 16384, "dim": 4096, "type": "bf16", "residual": True},
        # one env step of 8192 envs: norm to 8 bits, then the first projection of the block
        {"name": "q8 projection of 8192 envs", "op": "q8", "rows": 8192, "dim": 256, "out": 1024, "type": "bf16", "bias": False},
        # a single env: latency
        {"name": "i8 product, one token", "op": "i8", "rows": 1, "dim": 512, "out": 1000, "type": "f32", "bias": True},
        # the largest product: bound by the matrix cores
        {"name": "i8 product, 8192 cubed", "op": "i8", "rows": 8192, "dim": 8192, "out": 8192, "type": "bf16", "bias": False},
        # replay windows again, episodes ending inside them
        {"name": "conv windows f32", "op": "conv", "batch": 512, "length": 33, "dim": 512, "width": 4, "type": "f32",
         "silu": True, "starts": True},
        # two long sequences of an odd length, training in 16 bits
        {"name": "conv long bf16", "op": "conv", "batch": 2, "length": 8191, "dim": 2048, "width": 4, "type": "bf16",
         "silu": True, "starts": False},
        # one env step of 8192 envs
        {"name": "conv step of 8192 envs", "op": "conv_step", "batch": 8192, "dim": 512, "width": 4, "type": "f32"},
        {"name": "scan windows f32", "op": "scan", "batch": 512, "length": 33, "dim": 512, "state": 16, "groups": 1,
         "type": "f32", "gate": True, "starts": True, "train": True},
        # a long prompt of one sequence: few rows, work split over the length
        {"name": "scan prompt bf16", "op": "scan", "batch": 1, "length": 8192, "dim": 2048, "state": 16, "groups": 1,
         "type": "bf16", "gate": True, "starts": False, "train": False},
        # training on long sequences
        {"name": "scan long training bf16", "op": "scan", "batch": 4, "length": 2048, "dim": 2048, "state": 16,
         "groups": 1, "type": "bf16", "gate": True, "starts": False, "train": True},
        {"name": "scan step of 8192 envs", "op": "scan_step", "batch": 8192, "dim": 512, "state": 16, "groups": 1,
         "type": "f32"},
    ]


def _size(rng, lo, hi):
    """A whole number between lo and hi, evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "q8", "i8", "conv", "conv_step", "scan", "scan", "scan_step"])
    t = rng.choice(["f32", "bf16", "f16"])
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "norm":
        dim = _size(rng, 8, 8192)
        return {"op": op, "rows": _size(rng, 1, (1 << 25) // dim), "dim": dim, "type": t, "residual": yes()}
    if op == "q8":
        return {"op": op, "rows": _size(rng, 1, 8192), "dim": _size(rng, 16, 1024), "out": _size(rng, 16, 2048),
                "type": rng.choice(["bf16", "f16"]), "bias": yes()}
    if op == "i8":
        return {"op": op, "rows": _size(rng, 1, 8192), "dim": _size(rng, 16, 8192), "out": _size(rng, 16, 8192),
                "type": t, "bias": yes()}
    if op == "conv":
        length, dim = _size(rng, 1, 8192), _size(rng, 16, 2048)
        return {"op": op, "batch": _size(rng, 1, max(1, (1 << 24) // (length * dim))), "length": length, "dim": dim,
                "width": rng.choice([2, 3, 4]), "type": t, "silu": yes(), "starts": yes()}
    if op == "conv_step":
        return {"op": op, "batch": _size(rng, 1, 8192), "dim": _size(rng, 16, 512), "width": rng.choice([2, 3, 4]), "type": t}
    groups = rng.choice([1, 1, 2])
    dim = _size(rng, 8, 256) * groups
    state = rng.choice([4, 8, 16, 16])
    if op == "scan":
        length, train = _size(rng, 1, 4096), yes()
        return {"op": op, "batch": _size(rng, 1, max(1, (1 << 23) // (length * dim))), "length": length, "dim": dim,
                "state": state, "groups": groups, "type": t, "gate": yes(), "starts": yes(), "train": train}
    return {"op": op, "batch": _size(rng, 1, 8192), "dim": dim, "state": state, "groups": groups, "type": t}


def work(c):
    e = BYTES[c["type"]]
    if c["op"] == "norm":
        n = c["rows"] * c["dim"]
        r = 1 if c["residual"] else 0
        # x (+ residual), dy, ds in; y, (s), dx out; the weight's gradient
        return {"bytes": n * e * (5 + 2 * r) + 8 * c["dim"], "flops": 16.0 * n}
    if c["op"] == "q8":
        m, k, n = c["rows"], c["dim"], c["out"]
        return {"bytes": m * k * e * 3 + n * k + m * n * e + 4 * (n + k), "flops": 2.0 * m * n * k}
    if c["op"] == "i8":
        m, k, n = c["rows"], c["dim"], c["out"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e, "flops": 2.0 * m * n * k}
    if c["op"] == "conv":
        n = c["batch"] * c["length"] * c["dim"]
        return {"bytes": n * e * 4, "flops": n * (6.0 * c["width"] + 20)}
    if c["op"] == "conv_step":
        n = c["batch"] * c["dim"]
        return {"bytes": n * e * (2 + 2 * (c["width"] - 1)), "flops": n * (2.0 * c["width"] + 8)}
    g = c["groups"] * c["state"]
    if c["op"] == "scan":
        n, bl = c["batch"] * c["length"] * c["dim"], c["batch"] * c["length"]
        z = 1 if c["gate"] else 0
        k = c["batch"] * c["dim"] * c["state"] * 4
        if not c["train"]:
            return {"bytes": n * e * (3 + z) + 2 * bl * g * e + 2 * k, "flops": n * (6.0 * c["state"] + 12)}
        # y; then u, delta, (z), dout once, their gradients; B, C and theirs; the states at the ends and theirs
        return {"bytes": n * e * (6 + 2 * z) + 4 * bl * g * e + 4 * k, "flops": n * (24.0 * c["state"] + 40)}
    n = c["batch"] * c["dim"]
    return {"bytes": n * e * 4 + 2 * c["batch"] * g * e + 8 * n * c["state"], "flops": n * (6.0 * c["state"] + 12)}


# ---------------------------------------------------------------------------------- inputs
def _starts(g, batch, length):
    """Episodes end inside the windows now and then; 300 steps are the longest."""
    return (torch.rand(batch, length, device=DEV, generator=g) < 1.0 / 60).to(torch.uint8)


def _int8(g, rows, dim):
    q = (torch.randn(rows, dim, device=DEV, generator=g) * 32).round_().clamp_(-127, 127)
    return q.to(torch.int8), torch.rand(rows, device=DEV, generator=g) * 0.02 + 0.005


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[c["type"]]

    def rand(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)

    f32 = torch.float32
    s = {"case": c}
    if c["op"] == "norm":
        m, d = c["rows"], c["dim"]
        s.update(x=rand(m, d), r=rand(m, d) if c["residual"] else None, w=1 + rand(d, scale=0.1, dtype=f32),
                 dy=rand(m, d), ds=rand(m, d))
    elif c["op"] == "q8":
        m, d = c["rows"], c["dim"]
        q, scale = _int8(g, c["out"], d)
        s.update(x=rand(m, d), r=rand(m, d), w=1 + rand(d, scale=0.1, dtype=f32), wq=q, wscale=scale,
                 bias=rand(c["out"], dtype=f32) if c["bias"] else None)
    elif c["op"] == "i8":
        q, scale = _int8(g, c["rows"], c["dim"])
        wq, wscale = _int8(g, c["out"], c["dim"])
        s.update(q=q, scale=scale, wq=wq, wscale=wscale, bias=rand(c["out"], dtype=f32) if c["bias"] else None)
    elif c["op"] == "conv":
        b, n, d, w = c["batch"], c["length"], c["dim"], c["width"]
        s.update(x=rand(b, n, d), w=rand(d, w, scale=w ** -0.5, dtype=f32), bias=rand(d, scale=0.1, dtype=f32),
                 state=rand(b, w - 1, d), starts=_starts(g, b, n) if c["starts"] else None, dy=rand(b, n, d))
    elif c["op"] == "conv_step":
        b, d, w = c["batch"], c["dim"], c["width"]
        s.update(x=rand(b, d), w=rand(d, w, scale=w ** -0.5, dtype=f32), bias=rand(d, scale=0.1, dtype=f32),
                 state=rand(b, w - 1, d), reset=(torch.rand(b, device=DEV, generator=g) < 0.01).to(torch.uint8))
    else:
        b, d, n, k = c["batch"], c["dim"], c["state"], c["groups"]
        lead = (b, c["length"]) if c["op"] == "scan" else (b,)
        dt = torch.exp(torch.rand(d, device=DEV, generator=g) * math.log(100.0) + math.log(1e-3))   # 0.001 .. 0.1
        A = -torch.arange(1, n + 1, device=DEV, dtype=f32).repeat(d, 1) * (1 + 0.1 * torch.rand(d, n, device=DEV, generator=g))
        s.update(u=rand(*lead, d), delta=rand(*lead, d, scale=0.5), A=A, B=rand(*lead, k, n), C=rand(*lead, k, n),
                 D=1 + rand(d, scale=0.1, dtype=f32), bias=dt + torch.log(-torch.expm1(-dt)), h=rand(b, d, n, dtype=f32))
        if c["op"] == "scan":
            s.update(z=rand(*lead, d) if c["gate"] else None, starts=_starts(g, b, c["length"]) if c["starts"] else None,
                     dy=rand(*lead, d), dh=rand(b, d, n, dtype=f32))
        else:
            s.update(z=rand(*lead, d), reset=(torch.rand(b, device=DEV, generator=g) < 0.01).to(torch.uint8))
    return s


# ---------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    return _own(s, op) if own else PLAIN[op](s)


def _own(s, op):
    path = os.path.join(os.getcwd(), "mujoco-panda-pnp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from pnp_amd import seqops as ops

    leaf = lambda x: None if x is None else x.detach().requires_grad_(True)  # noqa: E731
    c = s["case"]
    if op == "norm":
        x, r, w = leaf(s["x"]), leaf(s["r"]), leaf(s["w"])
        y, t = ops.add_rms_norm(x, w, r, eps=EPS)
        if r is None:   # the stream goes on as x itself
            dx, dw = torch.autograd.grad([y, t], [x, w], [s["dy"], s["ds"]])
            return y.detach(), dx, dw
        dx, dr, dw = torch.autograd.grad([y, t], [x, r, w], [s["dy"], s["ds"]])
        return y.detach(), dx, dw, t.detach(), dr
    if op == "q8":
        q, scale, t = ops.add_rms_norm_q8(s["x"], s["w"], s["r"], eps=EPS)
        return ops.matmul_i8(q, scale, s["wq"], s["wscale"], bias=s["bias"], out_dtype=s["x"].dtype), scale, t
    if op == "i8":
        return ops.matmul_i8(s["q"], s["scale"], s["wq"], s["wscale"], bias=s["bias"], out_dtype=TYPES[c["type"]])
    if op == "conv":
        x, w, b, h = leaf(s["x"]), leaf(s["w"]), leaf(s["bias"]), leaf(s["state"])
        y, last = ops.causal_conv(x, w, b, activation="silu" if c["silu"] else None, starts=s["starts"], state=h)
        return (y.detach(), last.detach()) + torch.autograd.grad(y, [x, w, b, h], s["dy"])
    if op == "conv_step":
        y = ops.causal_conv_step(s["x"], s["state"], s["w"], s["bias"], activation="silu", reset=s["reset"])
        return y, s["state"]
    if op == "scan_step":
        y = ops.selective_scan_step(s["u"], s["h"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                    delta_bias=s["bias"], reset=s["reset"])
        return y, s["h"]
    if not c["train"]:
        return ops.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["bias"],
                                  starts=s["starts"], state=s["h"])
    v = {k: leaf(s[k]) for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "h")}
    y, last = ops.selective_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], D=v["D"], z=v["z"], delta_bias=v["bias"],
                                 starts=s["starts"], state=v["h"])
    grads = torch.autograd.grad([y, last], [x for x in v.values() if x is not None], [s["dy"], s["dh"]])
    return (y.detach(), last.detach()) + grads


def _plain_norm(s):
    x, r, w, f = s["x"], s["r"], s["w"], torch.float32
    t = x if r is None else x + r
    tf = t.to(f)
    rho = torch.rsqrt((tf * tf).mean(1, keepdim=True) + EPS)
    n = tf * rho
    y = (n * w).to(x.dtype)
    g = s["dy"].to(f)
    gw = g * w
    dx = (s["ds"].to(f) + rho * (gw - n * (gw * n).mean(1, keepdim=True))).to(x.dtype)
    dw = (g * n).sum(0)
    return (y, dx, dw) if r is None else (y, dx, dw, t, dx)


def _plain_q8(s):
    t = s["x"] + s["r"]
    tf = t.to(torch.float32)
    y = tf * torch.rsqrt((tf * tf).mean(1, keepdim=True) + EPS) * s["w"]
    scale = y.abs().amax(1) / 127
    q = torch.round(y / scale[:, None])
    out = (q @ s["wq"].to(torch.float32).t()) * scale[:, None] * s["wscale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(s["x"].dtype), scale, t


def _plain_i8(s):
    out = (s["q"].to(torch.float32) @ s["wq"].to(torch.float32).t()) * s["scale"][:, None] * s["wscale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(TYPES[s["case"]["type"]])


def _reach(starts, length, width, batch):
    """[batch, length, width] truth values: whether tap j of token t lies in the token's own sequence."""
    back = torch.arange(width - 1, -1, -1, device=DEV)
    if starts is None:
        return torch.ones(batch, length, width, dtype=torch.bool, device=DEV)
    at = torch.arange(length, device=DEV)
    begun = torch.where(starts != 0, at, -width).cummax(1).values
    return (at[None, :, None] - back) >= torch.where(begun < 0, -width, begun)[:, :, None]


def _plain_conv(s):
    c, f = s["case"], torch.float32
    b, n, d, k = c["batch"], c["length"], c["dim"], c["width"]
    xs = torch.cat([s["state"], s["x"]], 1).to(f)
    ok = _reach(s["starts"], n, k, b)
    taps = torch.stack([xs[:, j:j + n] * ok[:, :, j, None] for j in range(k)], 3)      # [b, n, d, k]
    pre = (taps * s["w"]).sum(3) + s["bias"]
    sig = torch.sigmoid(pre)
    y = (pre * sig if c["silu"] else pre).to(s["x"].dtype)
    g = s["dy"].to(f)
    if c["silu"]:
        g = g * (sig * (1 + pre * (1 - sig)))
    dxs = torch.zeros_like(xs)
    for j in range(k):
        dxs[:, j:j + n] += g * s["w"][:, j] * ok[:, :, j, None]
    dw = (taps * g[..., None]).sum((0, 1))
    last = torch.cat([s["state"], s["x"]], 1)[:, n:].contiguous()
    if s["starts"] is not None:    # what lies before the last start is not part of the sequence that goes on
        after = _reach(torch.cat([s["starts"], torch.zeros_like(s["starts"][:, :1])], 1), n + 1, k, b)[:, n, :k - 1]
        last = last * after[:, :, None]
    t = s["x"].dtype
    return y, last, dxs[:, k - 1:].to(t), dw, g.sum((0, 1)), dxs[:, :k - 1].to(t)


def _plain_conv_step(s):
    f = torch.float32
    s["state"].masked_fill_(s["reset"].bool()[:, None, None], 0)
    xs = torch.cat([s["state"], s["x"][:, None]], 1)
    pre = (xs.to(f) * s["w"].t()).sum(1) + s["bias"]
    s["state"].copy_(xs[:, 1:])
    return (pre * torch.sigmoid(pre)).to(s["x"].dtype), s["state"]


def _softplus(x):
    return torch.where(x > 0, x, 0) + torch.log1p(torch.exp(-x.abs()))


def _linear(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dimension 1, by doubling."""
    a, b, k, n = a.clone(), b.clone(), 1, a.shape[1]
    while k < n:
        b[:, k:] += a[:, k:] * b[:, :-k].clone()
        a[:, k:] *= a[:, :-k].clone()
        k *= 2
    return b


def _spread(x, d):
    """[..., groups, n] of each channel: [..., d, n]"""
    return x.to(torch.float32).repeat_interleave(d // x.shape[-2], -2)


def _plain_scan(s):
    c, f = s["case"], torch.float32
    d = c["dim"]
    u, raw = s["u"].to(f), s["delta"].to(f) + s["bias"]
    dt = _softplus(raw)
    B, C = _spread(s["B"], d), _spread(s["C"], d)
    a = torch.exp(dt[..., None] * s["A"])
    if s["starts"] is not None:
        a = a * (s["starts"] == 0)[:, :, None, None]
    b = (dt * u)[..., None] * B
    b[:, 0] += a[:, 0] * s["h"]
    h = _linear(a, b)
    del b
    y = (h * C).sum(3) + s["D"] * u
    z = None if s["z"] is None else s["z"].to(f)
    sig = None if z is None else torch.sigmoid(z)
    out = (y if z is None else y * (z * sig)).to(s["u"].dtype)
    last = h[:, -1].contiguous()
    if not c["train"]:
        return out, last
    dout = s["dy"].to(f)
    dy = dout if z is None else dout * (z * sig)
    src = dy[..., None] * C
    src[:, -1] += s["dh"]
    back = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _linear(back.flip(1), src.flip(1)).flip(1)
    del src, back
    ah = a * torch.cat([s["h"][:, None], h[:, :-1]], 1)
    gb = (g * B).sum(3)
    dA = (g * ah * dt[..., None]).sum((0, 1))
    ddt = (g * ah * s["A"]).sum(3) + u * gb
    draw_ = ddt * torch.sigmoid(raw)
    k = (c["batch"], c["length"], c["groups"], d // c["groups"], c["state"])
    dB = (g * (dt * u)[..., None]).view(k).sum(3)
    dC = (h * dy[..., None]).view(k).sum(3)
    t = s["u"].dtype
    grads = [(s["D"] * dy + dt * gb).to(t), draw_.to(t), dA, dB.to(t), dC.to(t), (dy * u).sum((0, 1))]
    if z is not None:
        grads.append((dout * y * (sig * (1 + z * (1 - sig)))).to(t))
    grads += [draw_.sum((0, 1)), a[:, 0] * g[:, 0]]
    return (out, last, *grads)


def _plain_scan_step(s):
    f, d = torch.float32, s["case"]["dim"]
    u, dt, z = s["u"].to(f), _softplus(s["delta"].to(f) + s["bias"]), s["z"].to(f)
    a = torch.exp(dt[..., None] * s["A"]) * (s["reset"] == 0)[:, None, None]
    s["h"].copy_(a * s["h"] + (dt * u)[..., None] * _spread(s["B"], d))
    y = (s["h"] * _spread(s["C"], d)).sum(2) + s["D"] * u
    return (y * (z * torch.sigmoid(z))).to(s["u"].dtype), s["h"]


PLAIN = {"norm": _plain_norm, "q8": _plain_q8, "i8": _plain_i8, "conv": _plain_conv, "conv_step": _plain_conv_step,
         "scan": _plain_scan, "scan_step": _plain_scan_step}


# ---------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    wide = {k: v.double().requires_grad_(True) if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    return EXACT[c["op"]](c, s, wide)


def _exact_norm(c, s, v):
    # the sum is held in the inputs' type: the norm reads what is stored
    t = v["x"] if v["r"] is None else (s["x"] + s["r"]).double().requires_grad_(True)
    y = t / (t.pow(2).mean(1, keepdim=True) + EPS).sqrt() * v["w"]
    dt, dw = torch.autograd.grad([y, t], [t, v["w"]], [s["dy"].double(), s["ds"].double()])
    return (y, dt, dw) if v["r"] is None else (y, dt, dw, t, dt)


def _exact_q8(c, s, v):
    t = (s["x"] + s["r"]).double()
    y = t / (t.pow(2).mean(1, keepdim=True) + EPS).sqrt() * v["w"].detach()
    scale = y.abs().max(1).values / 127
    out = torch.round(y / scale[:, None]).mm(s["wq"].double().t().contiguous()) * scale[:, None] * s["wscale"].double()
    return out if v["bias"] is None else out + v["bias"].detach(), scale, t


def _exact_i8(c, s, v):
    out = s["q"].double().mm(s["wq"].double().t().contiguous()) * s["scale"].double()[:, None] * s["wscale"].double()
    return out if v["bias"] is None else out + v["bias"].detach()


def _exact_conv(c, s, v):
    k, n = c["width"], c["length"]
    held = list(v["state"].unbind(1))     # the taps, oldest first
    tokens = v["x"].unbind(1)
    outs = []
    for i in range(n):
        if s["starts"] is not None:
            held = [h * (s["starts"][:, i:i + 1] == 0) for h in held]
        held = held + [tokens[i]]
        outs.append(sum(h * v["w"][:, j] for j, h in enumerate(held)) + v["bias"])
        held = held[1:]
    pre = torch.stack(outs, 1)
    y = torch.nn.functional.silu(pre) if c["silu"] else pre
    last = torch.stack(held, 1)
    return (y, last) + torch.autograd.grad(y, [v["x"], v["w"], v["bias"], v["state"]], s["dy"].double())


def _exact_conv_step(c, s, v):
    held = v["state"].detach() * (s["reset"] == 0)[:, None, None]
    taps = torch.cat([held, v["x"].detach()[:, None]], 1)
    pre = torch.einsum("bjd,dj->bd", taps, v["w"].detach()) + v["bias"].detach()
    return torch.nn.functional.silu(pre), taps[:, 1:]


def _exact_token(v, h, u, delta, B, C, z, keep, per):
    dt = torch.nn.functional.softplus(delta + v["bias"], threshold=40.0)
    B, C = B.repeat_interleave(per, 1), C.repeat_interleave(per, 1)
    if keep is not None:
        h = h * keep[:, None, None]
    h = torch.exp(dt[:, :, None] * v["A"]) * h + (dt * u)[:, :, None] * B
    y = (h * C).sum(2) + v["D"] * u
    return h, y if z is None else torch.nn.functional.silu(z) * y


def _exact_scan(c, s, v):
    h, outs, per = v["h"], [], c["dim"] // c["groups"]
    with torch.set_grad_enabled(c["train"]):
        # tokens first, one unbind each: a slice of a leaf per token would add a gradient of the whole at each
        cols = [x.unbind(1) if x is not None else [None] * c["length"] for x in (v["u"], v["delta"], v["B"], v["C"], v["z"])]
        for i in range(c["length"]):
            keep = None if s["starts"] is None else (s["starts"][:, i] == 0)
            h, y = _exact_token(v, h, *(x[i] for x in cols), keep, per)
            outs.append(y)
        out = torch.stack(outs, 1)
    if not c["train"]:
        return out, h
    names = [k for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "h") if v[k] is not None]
    return (out, h) + torch.autograd.grad([out, h], [v[k] for k in names], [s["dy"].double(), s["dh"].double()])


def _exact_scan_step(c, s, v):
    with torch.no_grad():
        h, y = _exact_token(v, v["h"], v["u"], v["delta"], v["B"], v["C"], v["z"], s["reset"] == 0, c["dim"] // c["groups"])
    return y, h


EXACT = {"norm": _exact_norm, "q8": _exact_q8, "i8": _exact_i8, "conv": _exact_conv, "conv_step": _exact_conv_step,
         "scan": _exact_scan, "scan_step": _exact_scan_step}
