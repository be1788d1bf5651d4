"""Sequence operators (pnp_amd.seqops, csrc/seq_*.hip) on the device against tests/seq_plain.py in 64
bits, with tolerances that count roundings (seq_plain.close)."""
import itertools

import pytest
import torch

import seq_plain as P

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda t: str(t).replace("torch.", "") if isinstance(t, torch.dtype) else None   # noqa: E731


@pytest.fixture(scope="module")
def S():
    assert torch.cuda.is_available()
    from pnp_amd import seqops
    return seqops


class Draw:
    """Inputs on the CPU in their type, and the same values in 64 bits and on the device."""

    def __init__(self, seed):
        self.g = torch.Generator().manual_seed(seed)

    def __call__(self, *shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g) * scale).to(dtype)

    def starts(self, *shape, p=0.2):
        return (torch.rand(*shape, generator=self.g) < p).to(torch.uint8)


def dev(t, grad=False):
    return None if t is None else t.cuda().requires_grad_(grad)


def wide(t):
    return None if t is None else t.double()


# ---------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 8), (5, 33), (7, 256), (2, 257), (66, 512), (3, 1000), (2, 2048), (3, 4096),
                                      (2, 8192), (2, 16400), (1, 2047), (300, 64)])
def test_norm_and_gradient(S, dtype, rows, dim):
    d = Draw(rows * 10000 + dim)
    for res_type in dict.fromkeys((None, dtype, torch.float32)):
        x, r, w = d(rows, dim, dtype=dtype), None if res_type is None else d(rows, dim, dtype=res_type), 1 + d(dim, scale=0.2)
        dy, ds = d(rows, dim, dtype=dtype), d(rows, dim, dtype=res_type or dtype)
        gx, gr, gw = dev(x, True), dev(r, r is not None), dev(w, True)
        y, s = S.add_rms_norm(gx, gw, gr, eps=1e-5)
        held = x if r is None else (x.float() + r.float()).to(r.dtype)   # one rounding of an fp32 sum
        assert torch.equal(s.detach().cpu(), held)
        ref, _ = P.norm(wide(held), wide(w), 1e-5)
        # the squares' sum: a chain of dim / 64 and the lanes' 8; halved by the root; 4 more
        k = dim / 128 + 10
        P.close(y, ref, ref.abs(), k, "y")
        grads = torch.autograd.grad([y, s], [t for t in (gx, gr, gw) if t is not None], [dev(dy), dev(ds)])
        dx, bdx, dw, bdw = P.norm_grad(wide(held), wide(w), 1e-5, wide(dy), wide(ds))
        P.close(grads[0], dx, bdx, 4 * k, "dx")
        if r is not None:
            P.close(grads[1], dx, bdx, 4 * k, "dresidual")
        P.close(grads[-1], dw, bdw, k + rows + 24, "dweight")


def test_norm_strides_shapes_and_missing_gradients(S):
    d = Draw(1)
    big, w = d(4, 6, 80), 1 + d(40, scale=0.1)
    for x in (big[:, :, 3:43], big[:, ::2, :40], big.transpose(0, 1)[:, :, 40:], big[..., ::2]):
        y, s = S.add_rms_norm(dev(big).as_strided(x.size(), x.stride(), x.storage_offset()), dev(w))
        ref, _ = P.norm(wide(x), wide(w), 1e-6)
        P.close(y, ref, ref.abs(), 12, "strided")
        assert tuple(s.shape) == tuple(x.shape)
    # gradients through one of the outputs alone, and a broadcast dy
    x, r = dev(d(5, 40), True), dev(d(5, 40), True)
    y, s = S.add_rms_norm(x, dev(w), r)
    gx, gr = torch.autograd.grad(s.sum(), [x, r], retain_graph=True)
    assert torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, gx)
    gx, = torch.autograd.grad(y.sum(), [x])
    held = wide((x + r).detach().cpu())
    dx, bdx, _, _ = P.norm_grad(held, wide(w), 1e-6, torch.ones(5, 40).double(), torch.zeros(5, 40).double())
    P.close(gx, dx, bdx, 50, "dy broadcast")
    for shape in ((0, 40), (3, 0, 40)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        wg = dev(w, True)
        y, _ = S.add_rms_norm(x, wg)
        gx, gw = torch.autograd.grad(y.sum(), [x, wg])
        assert y.shape == x.shape and gx.shape == x.shape and not gw.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,dim", [(1, 16), (9, 33), (4, 256), (3, 1000), (2, 4096), (2, 16400), (2, 20001)])
def test_norm_in_8_bits(S, dtype, rows, dim):
    d = Draw(dim)
    x, r, w = d(rows, dim, dtype=dtype), d(rows, dim, dtype=dtype), 1 + d(dim, scale=0.2)
    with torch.no_grad():
        q, scale, s = S.add_rms_norm_q8(dev(x), dev(w), dev(r))
    held = (x.float() + r.float()).to(dtype)
    assert torch.equal(s.cpu(), held) and q.dtype == torch.int8 and tuple(q.shape) == (rows, dim)
    ref, _ = P.norm(wide(held), wide(w), 1e-6)
    check_q8(q, scale, ref, dim / 128 + 12)


def check_q8(q, scale, ref, k):
    """scale within k roundings of max|ref| / 127; q within half a step (and those roundings) of ref / scale."""
    top = ref.abs().amax(-1) / 127
    P.close(scale, top, top, k, "scale")
    off = (q.double().cpu() - ref / top[..., None]).abs()
    assert off.max() <= 0.5 + 127 * 2 * k * P.E32
    assert (q.cpu().abs().amax(-1) == 127).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_rows_in_8_bits(S, dtype):
    d = Draw(3)
    for shape in ((5, 24), (2, 3, 100), (1, 9000), (3, 20001)):
        x = d(*shape, dtype=dtype)
        q, scale = S.quantize_rows(dev(x))
        check_q8(q, scale, wide(x), 4)
    x = torch.zeros(6, 32, dtype=dtype)
    x[1, 3], x[2, 4], x[3, 5], x[4] = float("nan"), float("inf"), -float("inf"), 1e-30 if dtype != torch.float16 else 0.0
    x[5, 0] = 1.0
    q, scale = S.quantize_rows(dev(x))
    q, scale = q.cpu(), scale.cpu()
    assert scale[0] == 0 and not q[0].any()
    assert torch.isnan(scale[1:4]).all() and not q[1:4].any()
    assert torch.isfinite(scale[4]) and q[5, 0] == 127 and not q[5, 1:].any()
    with torch.no_grad():
        q, scale, _ = S.add_rms_norm_q8(dev(x), torch.ones(32, device="cuda"))
    assert scale[0] == 0 and torch.isnan(scale[1:4]).all() and not q[:4].any()


# ---------------------------------------------------------------------------------- product
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 1000, 512), (3, 17, 15), (16, 64, 16), (33, 40, 100), (65, 130, 257), (128, 128, 128),
                                   (200, 300, 1000), (257, 512, 640), (500, 260, 2064), (64, 1024, 4096), (7, 4099, 129), (2100, 2060, 208),
                                   (4096, 1030, 1040), (1025, 4609, 16)])
def test_product(S, M, N, K):
    d = Draw(M + N + K)
    q = torch.randint(-128, 128, (M, K), generator=d.g, dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=d.g, dtype=torch.int8)
    s, ws, b = d(M).abs() + 0.01, d(N).abs() + 0.01, d(N)
    acc = q.double() @ w.double().t()
    scaled = acc * wide(s)[:, None] * wide(ws)
    for dtype, bias in itertools.product(TYPES, (None, b)):
        if dtype == torch.float16:
            s = s * 2.0 ** -12    # (sums of 16 000 products would overflow half precision)
            scaled = acc * wide(s)[:, None] * wide(ws)
        ref = scaled if bias is None else scaled + wide(bias)
        out = S.matmul_i8(dev(q), dev(s), dev(w), dev(ws), bias=dev(bias), out_dtype=dtype)
        assert out.dtype == dtype
        P.close(out, ref, scaled.abs() + wide(b).abs(), 4, f"{M} {N} {K} {dtype}")


def test_product_strides_and_extremes(S):
    d = Draw(5)
    big = torch.randint(-127, 128, (40, 300), generator=d.g, dtype=torch.int8)
    w = torch.randint(-127, 128, (50, 300), generator=d.g, dtype=torch.int8)
    one = torch.ones(50)
    for qs, ks in ((slice(0, 40), slice(7, 107)), (slice(0, 40, 2), slice(0, 128)), (slice(3, 4), slice(1, 300))):
        a, b = big[qs, ks], w[:, ks]
        out = S.matmul_i8(dev(big)[qs, ks], torch.ones(a.shape[0], device="cuda"), dev(w)[:, ks], dev(one))
        assert torch.equal(out.double().cpu(), a.double() @ b.double().t())
    q, s = S.quantize_rows(dev(d(3, 5, 33)))              # padded rows of a batch of two dimensions
    out = S.matmul_i8(q, s, q.reshape(15, 33), torch.ones(15, device="cuda"))
    ref = q.double().cpu().reshape(15, 33)
    P.close(out.reshape(15, 15), ref @ ref.t() * s.double().cpu().reshape(15, 1), (ref @ ref.t() * s.double().cpu().reshape(15, 1)).abs(), 3)
    row = dev(big)[:1].expand(6, 300)                     # a broadcast row
    assert torch.equal(S.matmul_i8(row, torch.ones(6, device="cuda"), dev(w), dev(one)).double().cpu(),
                       big[:1].double().expand(6, 300) @ w.double().t())
    full = torch.full((2, 131071), -128, dtype=torch.int8, device="cuda")   # the largest sum there is
    out = S.matmul_i8(full, torch.ones(2, device="cuda"), full, torch.ones(2, device="cuda"))
    assert torch.equal(out.cpu(), torch.full((2, 2), float(16384 * 131071)))
    assert S.matmul_i8(full[:0], torch.ones(0, device="cuda"), full, torch.ones(2, device="cuda")).shape == (0, 2)
    nan = torch.tensor([float("nan"), 1.0], device="cuda")                  # a row that was not finite stays so
    out = S.matmul_i8(torch.zeros(2, 16, dtype=torch.int8, device="cuda"), nan, torch.zeros(3, 16, dtype=torch.int8, device="cuda"),
                      torch.ones(3, device="cuda"))
    assert torch.isnan(out[0]).all() and not out[1].any()


# ---------------------------------------------------------------------------------- convolution
CONVS = [(1, 1, 8, 4), (2, 3, 5, 4), (3, 33, 16, 4), (2, 130, 24, 3), (2, 67, 40, 2), (1, 700, 8, 4), (5, 2, 64, 4), (40, 33, 520, 4),
         (2, 9, 33, 3), (1, 8, 64, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,L,D,W", CONVS)
def test_conv_and_gradient(S, dtype, B, L, D, W):
    d = Draw(B + L * 100 + D)
    for silu, starts, state, bias in ((True, True, True, True), (False, False, False, False), (True, False, True, False)):
        x, w, b = d(B, L, D, dtype=dtype), d(D, W, scale=0.5), d(D) if bias else None
        st = d(B, W - 1, D, dtype=dtype) if state else None
        at = d.starts(B, L) if starts else None
        dy, dl = d(B, L, D, dtype=dtype), d(B, W - 1, D, dtype=dtype)
        gx, gw, gb, gs = dev(x, True), dev(w, True), dev(b, bias), dev(st, state)
        y, last = S.causal_conv(gx, gw, gb, activation="silu" if silu else None, starts=dev(at), state=gs)
        ry, rlast, bnd, grads, bounds = P.conv(wide(x), wide(w), wide(b), silu, at, wide(st), wide(dy), wide(dl))
        assert torch.equal(last.detach().double().cpu(), rlast)
        # pre: W products and sums; sigmoid of it: 2 |pre| + 6 steps, and |pre| <= 8 here
        P.close(y, ry, bnd + ry.abs(), W + 24, "y")
        leaves = dict(x=gx, w=gw, b=gb, state=gs)
        leaves = {k: v for k, v in leaves.items() if v is not None}
        got = torch.autograd.grad([y, last], list(leaves.values()), [dev(dy), dev(dl)])
        for k, v in zip(leaves, got):
            # silu': sigmoid twice; the weights' sums: a chain over a run, then the runs
            P.close(v, grads[k], bounds[k], 2 * W + 60 + (B * L / 8 + 80 if k in "wb" else 0), k)


def test_conv_strides_and_parts(S):
    d = Draw(11)
    big, w = d(3, 40, 64), d(24, 4)
    at = d.starts(3, 40, p=0.1)
    for x in (big[:, :, 7:31], big[..., 32:56], big[:, ::2, :24], big[..., 1:49:2]):
        g = dev(big)
        gx = g.as_strided(x.size(), x.stride(), x.storage_offset())
        s = at[:, :x.shape[1]].contiguous()
        y, _ = S.causal_conv(gx, dev(w), starts=dev(s))
        ry, _, bnd = P.conv(wide(x), wide(w), None, False, s, None)
        P.close(y, ry, bnd, 8, "strided")
    # a sequence in parts, and token by token, is the sequence
    x, st = d(3, 40, 24), d(3, 3, 24)
    whole, wl = S.causal_conv(dev(x), dev(w), activation="silu", starts=dev(at), state=dev(st))
    state, outs = dev(st), []
    for lo, hi in ((0, 1), (1, 1), (1, 18), (18, 40)):
        y, state = S.causal_conv(dev(x)[:, lo:hi], dev(w), activation="silu", starts=dev(at)[:, lo:hi], state=state)
        outs.append(y)
    assert torch.equal(torch.cat(outs, 1), whole) and torch.equal(state, wl)
    state, outs = dev(st).clone(), []
    for t in range(40):
        outs.append(S.causal_conv_step(dev(x)[:, t], state, dev(w), activation="silu", reset=dev(at)[:, t].bool()))
    P.close(torch.stack(outs, 1), wide(whole.cpu()), wide(whole.cpu()).abs() + 1, 30, "steps")
    assert torch.equal(state, wl)
    e = torch.zeros(0, 40, 24, device="cuda", requires_grad=True)
    gw = dev(w, True)
    y, last = S.causal_conv(e, gw)
    assert y.shape == (0, 40, 24) and last.shape == (0, 3, 24)
    assert not torch.autograd.grad(y.sum(), gw)[0].any()
    x0, s0 = torch.zeros(2, 0, 24, device="cuda", requires_grad=True), dev(d(2, 3, 24), True)
    y, last = S.causal_conv(x0, gw, state=s0)
    assert torch.equal(last, s0)
    gs, gw2 = torch.autograd.grad((last * 2).sum(), [s0, gw])
    assert torch.equal(gs, torch.full_like(gs, 2.0)) and not gw2.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,D,W", [(1, 8, 4), (3, 5, 2), (70, 64, 3), (9, 513, 4)])
def test_conv_step(S, dtype, B, D, W):
    d = Draw(B)
    x, st, w, b, reset = d(B, D, dtype=dtype), d(B, W - 1, D, dtype=dtype), d(D, W, scale=0.5), d(D), d.starts(B, p=0.5)
    gs = dev(st)
    y = S.causal_conv_step(dev(x), gs, dev(w), dev(b), activation="silu", reset=dev(reset))
    ry, rl, bnd = P.conv(wide(x)[:, None], wide(w), wide(b), True, reset[:, None], wide(st))
    P.close(y[:, None], ry, bnd + ry.abs(), W + 24, "y")
    assert torch.equal(gs.double().cpu(), rl)


# ---------------------------------------------------------------------------------- scan
SCANS = [(1, 1, 1, 1, 1), (2, 5, 3, 2, 1), (2, 33, 16, 4, 2), (3, 40, 12, 8, 3), (2, 70, 64, 16, 1), (1, 130, 66, 16, 2), (2, 17, 10, 5, 1),
         (1, 45, 24, 20, 1), (2, 18, 8, 12, 1), (1, 20, 8, 32, 2), (1, 19, 6, 64, 1), (2, 31, 300, 3, 1), (1, 600, 4, 16, 1), (9, 33, 128, 16, 1)]


def scan_inputs(d, B, L, D, N, G, dtype, gate=True, starts=True, state=True, skip=True):
    return dict(u=d(B, L, D, dtype=dtype), delta=d(B, L, D, scale=0.7, dtype=dtype), A=-(d(D, N).abs() + 0.2) * 2,
                B=d(B, L, G, N, dtype=dtype), C=d(B, L, G, N, dtype=dtype), D=d(D) if skip else None,
                z=d(B, L, D, dtype=dtype) if gate else None, bias=d(D, scale=0.5) - 2 if skip else None,
                starts=d.starts(B, L, p=0.1) if starts else None, state=d(B, D, N) if state else None)


def plain_scan(v, **kw):
    w = {k: wide(t) if k != "starts" else t for k, t in v.items()}
    return P.scan(w["u"], w["delta"], w["A"], w["B"], w["C"], w["D"], w["z"], w["bias"], w["starts"], w["state"], **kw)


def run_scan(S, v):
    return S.selective_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], D=v["D"], z=v["z"], delta_bias=v["bias"], starts=v["starts"],
                            state=v["state"])


def check_scan(S, v, d, dtype, grads=True):
    B, L, D = v["u"].shape
    N = v["A"].shape[1]
    dout, dl = d(B, L, D, dtype=dtype), d(B, D, N)
    g = {k: dev(t, grads and k != "starts" and t is not None) for k, t in v.items()}
    out, last = run_scan(S, g)
    if not grads:
        ro, rl, eo, el = plain_scan(v)
    else:
        ro, rl, eo, el, rg, eg = plain_scan(v, dout=wide(dout), dlast=wide(dl))
    P.close(out, ro, eo, 1, "out")
    P.close(last, rl, el, 1, "last")
    if grads:
        leaves = {k: t for k, t in g.items() if t is not None and k != "starts"}
        got = torch.autograd.grad([out, last], list(leaves.values()), [dev(dout), dev(dl)])
        for k, t in zip(leaves, got):
            assert t.dtype == v[k].dtype
            P.close(t, rg[k], eg[k], 1, "d" + k)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,L,D,N,G", SCANS)
def test_scan_and_gradient(S, dtype, B, L, D, N, G):
    d = Draw(B * 1000 + L)
    check_scan(S, scan_inputs(d, B, L, D, N, G, dtype), d, dtype)


@pytest.mark.parametrize("gate,starts,state,skip", list(itertools.product([False, True], repeat=4)))
def test_scan_options(S, gate, starts, state, skip):
    d = Draw(77)
    check_scan(S, scan_inputs(d, 2, 37, 20, 6, 2, torch.float32, gate, starts, state, skip), d, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("starts", [False, True])
def test_scan_long_and_cut_in_chunks(S, dtype, starts):
    d = Draw(5)
    v = scan_inputs(d, 1, 1500, 72, 16, 1, dtype, starts=starts)
    if starts:
        v["starts"] = d.starts(1, 1500, p=0.002)
    check_scan(S, v, d, dtype)


def test_scan_every_token_a_start_and_dt_extremes(S):
    d = Draw(6)
    v = scan_inputs(d, 2, 20, 8, 4, 1, torch.float32)
    v["starts"] = torch.ones(2, 20, dtype=torch.uint8)
    check_scan(S, v, d, torch.float32)
    v = scan_inputs(d, 2, 20, 8, 4, 1, torch.float32)
    v["delta"] = d(2, 20, 8, scale=12.0)        # softplus from 1e-16 to 40
    check_scan(S, v, d, torch.float32)
    v["A"] = v["A"].abs() * 0.01                # growing states
    v["delta"] = d(2, 20, 8)
    check_scan(S, v, d, torch.float32)


def test_scan_sees_nothing_from_before_a_start(S):
    """Infinity and NaN before a start, in the state as in the tokens, do not reach what follows, forward or back."""
    d = Draw(8)
    v = scan_inputs(d, 2, 40, 12, 16, 1, torch.float32)
    v["starts"] = torch.zeros(2, 40, dtype=torch.uint8)
    v["starts"][0, 0] = v["starts"][1, 20] = 1
    clean = {k: dev(t) for k, t in v.items()}
    bad = {k: None if t is None else t.clone() for k, t in clean.items()}
    bad["state"][0] = float("nan")
    bad["state"][1, 3] = float("inf")
    bad["u"][1, 5] = float("inf")
    bad["u"][1, 19, 2] = float("nan")
    a, la = run_scan(S, clean)
    b, lb = run_scan(S, bad)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1, 20:], b[1, 20:]) and torch.equal(la, lb)
    assert torch.isnan(b[1, 19]).any()
    gb = {k: t if t is None or k == "starts" else t.clone().requires_grad_(True) for k, t in bad.items()}
    ga = {k: t if t is None or k == "starts" else t.clone().requires_grad_(True) for k, t in clean.items()}
    dout = torch.zeros(2, 40, 12, device="cuda")
    dout[0], dout[1, 20:] = 1.0, 1.0
    names = ("u", "delta", "B", "C", "z")
    da = torch.autograd.grad(run_scan(S, ga)[0], [ga[k] for k in names], dout)
    db = torch.autograd.grad(run_scan(S, gb)[0], [gb[k] for k in names], dout)
    for k, x, y in zip(names, da, db):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1, 20:], y[1, 20:]), k
    x, xs, w = dev(d(2, 9, 8)), dev(d(2, 3, 8)), dev(d(8, 4))
    at = torch.zeros(2, 9, dtype=torch.uint8, device="cuda")
    at[:, 4] = 1
    y, last = S.causal_conv(x, w, starts=at, state=xs)
    x2, xs2 = x.clone(), xs.clone()
    x2[:, :4], xs2[:] = float("nan"), float("inf")
    y2, last2 = S.causal_conv(x2, w, starts=at, state=xs2)
    assert torch.equal(y[:, 4:], y2[:, 4:]) and torch.equal(last, last2)


def test_scan_strides_parts_and_steps(S):
    d = Draw(9)
    B, L, D, N = 3, 50, 24, 16
    proj, xp, w = d(B, L, 2 * D + 8), d(B, L, 7 + 2 * N), scan_inputs(d, B, L, D, N, 1, torch.float32)
    gp, gx = dev(proj), dev(xp)
    v = {**{k: dev(t) for k, t in w.items()}, "u": gp[..., :D], "z": gp[..., D:2 * D], "B": gx[..., 7:7 + N, ], "C": gx[..., 7 + N:]}
    ref = {**w, "u": proj[..., :D], "z": proj[..., D:2 * D], "B": xp[..., None, 7:7 + N], "C": xp[..., None, 7 + N:]}
    out, last = run_scan(S, v)
    ro, rl, eo, el = plain_scan(ref)
    P.close(out, ro, eo, 1, "strided")
    P.close(last, rl, el, 1, "last")
    state, parts = v["state"], []
    for lo, hi in ((0, 1), (1, 1), (1, 30), (30, 50)):
        cut = {k: t[:, lo:hi] if k in ("u", "delta", "z", "B", "C", "starts") else t for k, t in v.items()}
        y, state = run_scan(S, {**cut, "state": state})
        parts.append(y)
    P.close(torch.cat(parts, 1), ro, eo, 1, "parts")
    P.close(state, rl, el, 1, "state of the parts")
    state, steps = v["state"].clone(), []
    for t in range(L):
        steps.append(S.selective_scan_step(v["u"][:, t], state, v["delta"][:, t], v["A"], v["B"][:, t], v["C"][:, t], D=v["D"], z=v["z"][:, t],
                                           delta_bias=v["bias"], reset=v["starts"][:, t]))
    P.close(torch.stack(steps, 1), ro, eo, 1, "steps")
    P.close(state, rl, el, 1, "state of the steps")
    with pytest.raises(ValueError, match="contiguous"):
        S.selective_scan_step(v["u"][:, 0], state.transpose(1, 2).contiguous().transpose(1, 2), v["delta"][:, 0], v["A"], v["B"][:, 0], v["C"][:, 0])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (5, 12, 16, 2), (3, 10, 5, 1), (70, 64, 16, 1), (3, 8, 12, 1), (2, 6, 64, 3), (4, 9, 32, 1)])
def test_scan_step(S, dtype, B, D, N, G):
    d = Draw(B + D)
    v = scan_inputs(d, B, 1, D, N, G, dtype)
    v["starts"] = d.starts(B, 1, p=0.4)
    g = {k: dev(t) for k, t in v.items()}
    ro, rl, eo, el = plain_scan(v)
    out = S.selective_scan_step(g["u"][:, 0], g["state"], g["delta"][:, 0], g["A"], g["B"][:, 0], g["C"][:, 0], D=g["D"], z=g["z"][:, 0],
                                delta_bias=g["bias"], reset=g["starts"][:, 0])
    P.close(out[:, None], ro, eo, 1, "out")
    P.close(g["state"], rl, el, 1, "state")


def test_scan_step_of_more_states_than_the_cache_holds(S):
    """The way past the caches gives the bits of the way through them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    B, D, N = 6272, 512, 16
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    u, dl, z, Bm, Cm, A, h = rnd(B, D), rnd(B, D), rnd(B, D), rnd(B, N), rnd(B, N), -rnd(D, N).abs(), rnd(B, D, N)
    assert h.numel() >= 50 * 1000 * 1000
    part, outs = [h[k:k + 448].clone() for k in range(0, B, 448)], []
    whole = S.selective_scan_step(u, h, dl, A, Bm, Cm, z=z)
    for i, p in enumerate(part):
        k = slice(448 * i, 448 * i + 448)
        outs.append(S.selective_scan_step(u[k], p, dl[k], A, Bm[k], Cm[k], z=z[k]))
    assert torch.equal(whole, torch.cat(outs)) and torch.equal(h, torch.cat(part))


def test_scan_empty(S):
    d = Draw(2)
    v = {k: dev(t, k != "starts") for k, t in scan_inputs(d, 2, 4, 8, 4, 1, torch.float32).items()}
    none = {k: t[:0] if k not in ("A", "D", "bias") else t for k, t in v.items()}
    out, last = run_scan(S, none)
    assert out.shape == (0, 4, 8) and last.shape == (0, 8, 4)
    ga, gd = torch.autograd.grad(out.sum() + last.sum(), [v["A"], v["D"]])
    assert not ga.any() and not gd.any()
    short = {k: t[:, :0] if k not in ("A", "D", "bias", "state") else t for k, t in v.items()}
    out, last = run_scan(S, short)
    assert out.shape == (2, 0, 8) and torch.equal(last, v["state"])
    gs, ga = torch.autograd.grad((3 * last).sum(), [v["state"], v["A"]])
    assert torch.equal(gs, torch.full_like(gs, 3.0)) and not ga.any()


# ---------------------------------------------------------------------------------- against differences
def test_gradients_against_differences(S):
    """A directional difference of the kernels' own forward, fp32, h = 2^-6: off by h^2 / 6 of the third derivative along
    the way (of the order of the loss, whose terms are smooth at scale 1: 1e-4) and by roundings / h of the loss's sum of
    magnitudes, which are random: 2^-24 * 64 * |terms| / sqrt(n)."""
    d = Draw(4)
    v = scan_inputs(d, 2, 24, 16, 8, 2, torch.float32)
    g = {k: dev(t) for k, t in v.items()}
    dout = dev(d(2, 24, 16))
    names = ("u", "delta", "A", "B", "C", "D", "z", "bias", "state")
    cases = [(names, g, lambda v: run_scan(S, v)[0], dout)]
    c = dict(x=dev(d(2, 24, 16)), w=dev(d(16, 4)), b=dev(d(16)), state=dev(d(2, 3, 16)))
    cases.append((tuple(c), c, lambda v: S.causal_conv(v["x"], v["w"], v["b"], activation="silu", starts=g["starts"], state=v["state"])[0], dout))
    n = dict(x=dev(d(48, 16)), r=dev(d(48, 16)), w=dev(d(16)))
    cases.append((tuple(n), n, lambda v: S.add_rms_norm(v["x"], v["w"], v["r"])[0], dout.reshape(48, 16)))
    for names, v, f, dy in cases:
        leaves = {k: t if k not in names else t.clone().requires_grad_(True) for k, t in v.items()}
        grads = torch.autograd.grad(f(leaves), [leaves[k] for k in names], dy)
        for k, grad in zip(names, grads):
            way = dev(d(*v[k].shape))
            way = way / way.norm()
            h = 2.0 ** -6
            with torch.no_grad():
                hi, lo = (f({**v, k: v[k] + s * h * way}).double() for s in (1, -1))
            diff = ((hi - lo) * dy.double()).sum() / (2 * h)
            want = (grad.double() * way.double()).sum()
            assert abs(diff - want) < 2e-3 * (1 + abs(want) + grad.double().norm() * 0.1), (k, float(diff), float(want))


# ---------------------------------------------------------------------------------- streams, graphs, repeats, refusals
def all_ops(S, v, x, w, q):
    """A pass through every operator on the same tensors."""
    y, s = S.add_rms_norm(v["u"], torch.ones_like(v["D"]), v["z"])
    c, cl = S.causal_conv(y, w, activation="silu", starts=v["starts"])
    o, last = run_scan(S, {**v, "u": c})
    grads = torch.autograd.grad([o, s], [v["u"], v["delta"], v["A"], v["B"], v["z"]], [v["delta"].detach(), v["u"].detach()]) if v["u"].requires_grad else ()
    with torch.no_grad():
        n8, sc, _ = S.add_rms_norm_q8(v["u"].detach(), torch.ones_like(v["D"]), v["z"].detach())
        p = S.matmul_i8(n8, sc, *q)
    return (y, c, cl, o, last, p) + grads


def op_inputs(S, seed, grad):
    d = Draw(seed)
    v = {k: dev(t, grad and k != "starts") for k, t in scan_inputs(d, 2, 300, 64, 16, 1, torch.float32).items()}
    return v, None, dev(d(64, 4)), S.quantize_rows(dev(d(40, 64)))


def test_repeats_are_bitwise_equal_and_streams_do_not_meet(S):
    sets = [op_inputs(S, k, True) for k in range(3)]
    want = [all_ops(S, *s) for s in sets]
    torch.cuda.synchronize()
    again = [all_ops(S, *s) for s in sets]
    for a, b in zip(want, again):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None] * 3
    for _ in range(3):
        for k, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[k] = all_ops(S, *sets[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_graphs_replay_as_eager(S):
    """Two captured graphs of every operator, forward and back, replayed in turn with eager work between."""
    sets = [op_inputs(S, k, True) for k in (10, 11)]
    graphs, outs = [], []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                all_ops(S, *s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(all_ops(S, *s))
        graphs.append(g)
    for k in range(6):
        with torch.no_grad():
            for s in sets:
                s[0]["u"].add_(0.01)      # new inputs at the same place
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        held = [[t.clone() for t in o] for o in outs]
        for s, o in zip(sets, held):
            eager = all_ops(S, *s)
            assert all(torch.equal(x, y) for x, y in zip(o, eager)), k


def test_refusals_on_the_device(S):
    x = torch.zeros(2, 3, 8, device="cuda")
    A, B, w = -torch.ones(8, 4, device="cuda"), torch.zeros(2, 3, 4, device="cuda"), torch.ones(8, 4, device="cuda")
    i8 = torch.zeros(2, 16, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    for error, call in [
        (TypeError, lambda: S.add_rms_norm(x.double(), w[:, 0])), (ValueError, lambda: S.add_rms_norm(x, w)),
        (ValueError, lambda: S.add_rms_norm(x, w[:, 0], x[:1])), (TypeError, lambda: S.add_rms_norm(x, w[:, 0], x.bfloat16())),
        (ValueError, lambda: S.add_rms_norm(x, w[:, 0], eps=-1.0)), (ValueError, lambda: S.add_rms_norm(x, w[:, 0].cpu())),
        (TypeError, lambda: S.add_rms_norm(x, None)),
        (TypeError, lambda: S.matmul_i8(i8.int(), one, i8, one)), (ValueError, lambda: S.matmul_i8(i8[:, :8], one, i8, one)),
        (ValueError, lambda: S.matmul_i8(i8, one[:1], i8, one)), (TypeError, lambda: S.matmul_i8(i8, one, i8, one, out_dtype=torch.float64)),
        (ValueError, lambda: S.causal_conv(x, torch.ones(8, 5, device="cuda"))), (ValueError, lambda: S.causal_conv(x, w[:4])),
        (ValueError, lambda: S.causal_conv(x, w, activation="relu")), (ValueError, lambda: S.causal_conv(x[0], w)),
        (TypeError, lambda: S.causal_conv(x, w, starts=torch.zeros(2, 3, device="cuda"))),
        (ValueError, lambda: S.causal_conv(x, w, starts=torch.zeros(2, 2, dtype=torch.bool, device="cuda"))),
        (TypeError, lambda: S.causal_conv(x, w, state=torch.zeros(2, 3, 8, dtype=torch.bfloat16, device="cuda"))),
        (ValueError, lambda: S.causal_conv(x, w, state=torch.zeros(2, 2, 8, device="cuda"))),
        (ValueError, lambda: S.selective_scan(x, x[:, :2], A, B, B)), (ValueError, lambda: S.selective_scan(x, x, A[:, 0], B, B)),
        (ValueError, lambda: S.selective_scan(x, x, A, B, B[..., :3])), (TypeError, lambda: S.selective_scan(x, x.half(), A, B, B)),
        (ValueError, lambda: S.selective_scan(x, x, A, torch.zeros(2, 3, 3, 4, device="cuda"), torch.zeros(2, 3, 3, 4, device="cuda"))),
        (TypeError, lambda: S.selective_scan(x, x, A, B, B, state=torch.zeros(2, 8, 4, dtype=torch.bfloat16, device="cuda"))),
        (ValueError, lambda: S.selective_scan(x, x, A, B, B, state=torch.zeros(2, 4, 8, device="cuda"))),
        (ValueError, lambda: S.selective_scan(x, x, -torch.ones(8, 65, device="cuda"), B, B)),
    ]:
        with pytest.raises(error):
            call()
