"""The sequence operators in 64 bits, token by token, for the tests of pnp_amd.seqops: values,
gradients by the formulas, and how far fp32 arithmetic can be off.

``Bound`` tensors hold the same formulas with every term's magnitude: sums of magnitudes, through which
no cancellation makes a result smaller than its terms.  A result of K roundings along its longest chain
is then off by at most K * 2^-24 * Bound (first order), plus half a step of the type it is stored in."""
import torch

STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # half a step below the normals
E32 = 2.0 ** -24


def close(got, ref, bound, roundings, name=""):
    """|got - ref| <= half a step of got's type + roundings * 2^-24 * bound, everywhere (NaN and infinity alike)."""
    assert tuple(got.shape) == tuple(ref.shape), (name, got.shape, ref.shape)
    g, ref, bound = got.detach().double().cpu(), ref.detach().double().cpu(), bound.detach().double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), name
    assert torch.equal(g[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), name
    off = (g - ref).abs()[fine]
    # rounding the off result: half a step of a value that may itself be off
    slack = roundings * E32 * bound[fine]
    tol = slack + STEP[got.dtype] * (ref.abs()[fine] + slack) + TINY[got.dtype]
    if off.numel():
        worst = (off / tol).max()
        assert worst <= 1, f"{name}: {float(worst):.3g} times the tolerance, off by {float(off.max()):.3g}"


def sig(x):
    return 1 / (1 + torch.exp(-x))


def softplus(x):
    return x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))


# ---------------------------------------------------------------------------------- norm
def norm(s, w, eps):
    rho = 1 / ((s * s).mean(-1, keepdim=True) + eps).sqrt()
    return s * rho * w, rho


def norm_grad(s, w, eps, dy, ds):
    """dx, its bound, dw, its bound"""
    _, rho = norm(s, w, eps)
    n, g = s * rho, dy * w
    dx = ds + rho * (g - n * (g * n).mean(-1, keepdim=True))
    bdx = ds.abs() + rho * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    return dx, bdx, (dy * n).sum(0), (dy * n).abs().sum(0)


# ---------------------------------------------------------------------------------- convolution
def conv(x, w, b, silu, starts, state, dy=None, dlast=None):
    """y, last, bound of y; with dy: a dict of gradients and one of their bounds"""
    B, L, D = x.shape
    W = w.shape[1]
    keep = torch.ones(B, L, dtype=torch.bool) if starts is None else starts == 0
    xs = torch.cat([torch.zeros(B, W - 1, D, dtype=x.dtype) if state is None else state, x], 1)

    def alive(t):   # [B, W]: tap j of token t (t = L: of the token after the last) is in its sequence
        out = torch.ones(B, W, dtype=torch.bool)
        for j in range(W - 2, -1, -1):
            # tap j reaches token t - (W - 1 - j): dropped if any token after it, up to t, starts
            at = t - (W - 1 - j) + 1
            out[:, j] = out[:, j + 1] & (keep[:, at] if 0 <= at < L else True)
        return out

    pre, bnd, reach = torch.zeros_like(x), torch.zeros_like(x), []
    for t in range(L):
        a = alive(t)
        reach.append(a)
        for j in range(W):
            tap = xs[:, t + j] * w[:, j]
            tap = torch.where(a[:, j, None], tap, torch.zeros_like(tap))
            pre[:, t] += tap
            bnd[:, t] += tap.abs()
    if b is not None:
        pre, bnd = pre + b, bnd + b.abs()
    y = pre * sig(pre) if silu else pre
    a = alive(L)
    last = torch.stack([torch.where(a[:, j, None], xs[:, L + j], torch.zeros_like(xs[:, L + j])) for j in range(W - 1)], 1)
    if dy is None:
        return y, last, bnd
    g = dy * (sig(pre) * (1 + pre * (1 - sig(pre)))) if silu else dy
    # |silu'| <= 1.1, |silu''| <= 0.5: an error of pre moves g by half of it
    gb = dy.abs() * (1.1 + 0.5 * bnd) if silu else dy.abs()
    dxs, bxs = torch.zeros_like(xs), torch.zeros_like(xs)
    dw, bw = torch.zeros_like(w), torch.zeros_like(w)
    for t in range(L):
        for j in range(W):
            m = reach[t][:, j, None]
            dxs[:, t + j] += torch.where(m, g[:, t] * w[:, j], torch.zeros_like(g[:, t]))
            bxs[:, t + j] += torch.where(m, (gb[:, t] * w[:, j]).abs(), torch.zeros_like(g[:, t]))
            tap = torch.where(m, xs[:, t + j], torch.zeros_like(xs[:, t + j]))
            dw[:, j] += (g[:, t] * tap).sum(0)
            bw[:, j] += (gb[:, t] * tap.abs()).sum(0)
    if dlast is not None:
        for j in range(W - 1):
            dxs[:, L + j] += torch.where(a[:, j, None], dlast[:, j], torch.zeros_like(dlast[:, j]))
            bxs[:, L + j] += dlast[:, j].abs()
    grads = dict(x=dxs[:, W - 1:], w=dw, b=g.sum((0, 1)), state=dxs[:, :W - 1])
    bounds = dict(x=bxs[:, W - 1:], w=bw, b=gb.sum((0, 1)), state=bxs[:, :W - 1])
    return y, last, bnd, grads, bounds


# ---------------------------------------------------------------------------------- scan
def scan(u, delta, A, Bm, Cm, D=None, z=None, bias=None, starts=None, state=None, dout=None, dlast=None):
    """out, last and how far fp32 may be off them, in steps of 2^-24; with dout: a dict of gradients and one of
    their errors.  Bm, Cm [B, L, G, N].

    Errors, relative, in steps: dt = softplus(raw): exp2's argument |raw| * 1.5 and its own 2, log1p 2, the sum 1:
    |raw| 2 + 5 (an argument's absolute error is the exponential's relative one).  a = exp2(dt A2): the argument's
    relative error dt's + 2 (A2, the product), so kappa = |dt A| (2 |raw| + 8) + 2.  z sigmoid(z): 2 |z| + 6.
    A sum of n terms adds its longest chain of additions.  The recurrences carry their errors on as they carry
    their values; *B: sums of magnitudes."""
    B, L, d = u.shape
    N, G = A.shape[1], Bm.shape[2]
    per = d // G
    raw = delta if bias is None else delta + bias
    dt = softplus(raw)
    wide = lambda t: t.repeat_interleave(per, 2)   # noqa: E731
    Bw, Cw = wide(Bm), wide(Cm)
    a = torch.exp(dt[..., None] * A)
    edt = 2 * raw.abs() + 6
    kappa = (dt[..., None] * A).abs() * (edt[..., None] + 2) + 3
    keep = torch.ones(B, L, dtype=torch.bool) if starts is None else starts == 0
    zero = torch.zeros(B, d, N, dtype=u.dtype)
    h = zero if state is None else state
    hb, he = h.abs(), zero
    hs, hbs, hes, hp, hpb, hpe = [], [], [], [], [], []     # hp: what a token's decay was applied to
    for t in range(L):
        m = keep[:, t, None, None]
        for to, v in ((hp, h), (hpb, hb), (hpe, he)):
            to.append(torch.where(m, v, zero))
        term = (dt[:, t] * u[:, t])[..., None] * Bw[:, t]
        h, hb = a[:, t] * hp[-1] + term, a[:, t] * hpb[-1] + term.abs()
        he = a[:, t] * (hpe[-1] + kappa[:, t] * hpb[-1]) + term.abs() * (edt[:, t, :, None] + 3) + hb
        hs.append(h), hbs.append(hb), hes.append(he)
    st = lambda v: torch.stack(v, 1) if v else torch.zeros(B, 0, d, N, dtype=u.dtype)   # noqa: E731
    H, HB, HE, HP, HPB, HPE = st(hs), st(hbs), st(hes), st(hp), st(hpb), st(hpe)
    y, yb, ye = (H * Cw).sum(3), (HB * Cw.abs()).sum(3), (HE * Cw.abs()).sum(3)
    if D is not None:
        y, yb = y + D * u, yb + (D * u).abs()
    ye = ye + 9 * yb                                   # a product, 4 + log2(lanes) additions, the last one
    gate = torch.ones_like(u) if z is None else z * sig(z)
    egate = torch.zeros_like(u) if z is None else 2 * z.abs() + 7
    out, oute = y * gate, (ye + yb * (egate + 1)) * gate.abs()
    if dout is None:
        return out, h, oute, he
    dy = dout * gate
    g = zero if dlast is None else dlast
    gb, ge = g.abs(), zero
    gs, gbs, ges = [], [], []
    for t in range(L - 1, -1, -1):
        new = Cw[:, t] * dy[:, t, :, None]
        g, gb = g + new, gb + new.abs()
        ge = ge + new.abs() * (egate[:, t, :, None] + 2) + gb
        gs.append(g), gbs.append(gb), ges.append(ge)
        m = keep[:, t, None, None]
        ge = torch.where(m, a[:, t] * (ge + kappa[:, t] * gb), zero)
        g, gb = torch.where(m, a[:, t] * g, zero), torch.where(m, a[:, t] * gb, zero)
    GS, GB, GE = st(gs[::-1]), st(gbs[::-1]), st(ges[::-1])
    AH, AHB, AHE = a * HP, a * HPB, a * (HPE + kappa * HPB)
    s1, s1b, s1e = (GS * Bw).sum(3), (GB * Bw.abs()).sum(3), ((GE + 8 * GB) * Bw.abs()).sum(3)
    gah, gahb, gahe = GS * AH, GB * AHB, GE * AHB + GB * AHE + 2 * GB * AHB
    s2, s2b, s2e = (gah * A).sum(3), (gahb * A.abs()).sum(3), ((gahe + 8 * gahb) * A.abs()).sum(3)
    ddt, ddtb, ddte = s2 + u * s1, s2b + u.abs() * s1b, s2e + u.abs() * s1e + 2 * (s2b + u.abs() * s1b)
    sr = sig(raw)
    dr, drb, dre = ddt * sr, ddtb * sr, (ddte + ddtb * edt) * sr
    k = (B, L, G, per, N)
    dtu = (dt * u)[..., None]
    # sums over tokens: a chunk's in a chain, then the rows of chunks by sixteenths; over channels: lanes, waves, workgroups
    rows, cols = L + B / 16 + 24, 24 + per / 16
    w = dt[..., None]
    grads = dict(u=dt * s1, delta=dr, A=(gah * w).sum((0, 1)), B=(GS * dtu).view(k).sum(3),
                 C=(H * dy[..., None]).view(k).sum(3), bias=dr.sum((0, 1)), state=g)
    errs = dict(u=dt * (s1e + s1b * (edt + 2)), delta=dre,
                A=((gahe + gahb * (edt[..., None] + 1)) * w).sum((0, 1)) + rows * (gahb * w).sum((0, 1)),
                B=((GE + GB * (edt[..., None] + 3 + cols)) * dtu.abs()).view(k).sum(3),
                C=((HE + HB * (egate[..., None] + 2 + cols)) * dy.abs()[..., None]).view(k).sum(3),
                bias=(dre + rows * drb).sum((0, 1)), state=ge)
    if D is not None:
        grads["u"], errs["u"] = grads["u"] + D * dy, errs["u"] + (D * dy).abs() * (egate + 4)
        grads["D"], errs["D"] = (dy * u).sum((0, 1)), ((dy * u).abs() * (egate + 2 + rows)).sum((0, 1))
    errs["u"] = errs["u"] + grads["u"].abs()
    if z is not None:
        sz = sig(z)
        dg, dgb = sz * (1 + z * (1 - sz)), sz * (1 + z.abs() * (1 - sz))
        # 1 - sigmoid loses what the sigmoid is off by: (2 |z| + 6) sigmoid, absolute
        grads["z"] = dout * y * dg
        errs["z"] = dout.abs() * (ye * dg.abs() + yb * (dgb * (egate + 6) + sz * z.abs() * sz * egate))
    return out, h, oute, he, grads, errs
