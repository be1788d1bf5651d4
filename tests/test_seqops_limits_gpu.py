"""Calls of the sequence operators (pnp_amd.seqops) that their documentation allows at its edges: offsets past 32 bits,
the same tensor twice, broadcast and negated views, states that autograd or a graph holds, growing states."""
import pytest
import torch

import seq_plain as P
import test_seqops_gpu as T
from test_seqops_gpu import S, Draw, dev, plain_scan, run_scan, scan_inputs   # noqa: F401  (S: the fixture)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def near(a, b, steps):
    """Steps of a 16-bit type, or of a few roundings in fp32: another variant of a kernel, its products fused otherwise."""
    step = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[a.dtype]
    a, b = a.double(), b.double()
    assert ((a - b).abs() <= steps * step * b.abs().clamp_min(b.abs().mean())).all()


# ---------------------------------------------------------------------------------- autograd
def test_second_gradients_are_refused(S):
    x, w = dev(Draw(1)(2, 9, 16), True), torch.ones(16, 4, device="cuda")
    B = dev(Draw(2)(2, 9, 4))
    for y in (S.add_rms_norm(x, w[:, 0])[0], S.add_rms_norm(x, w[:, 0], x)[1], S.causal_conv(x, w)[0],
              S.selective_scan(x, x, -w, B, B)[0]):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="second gradient"):
            g.sum().backward()


def test_a_state_advanced_in_place_is_refused_by_the_graph_that_holds_it(S):
    d = Draw(3)
    x, w, A, B = dev(d(2, 5, 8), True), dev(d(8, 4)), -torch.ones(8, 4, device="cuda"), dev(d(2, 5, 4))
    conv, ssm = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
    y, _ = S.causal_conv(x, w, state=conv)
    o, _ = S.selective_scan(x, x, A, B, B, state=ssm)
    with torch.no_grad():
        S.causal_conv_step(x[:, 0], conv, w)
        S.selective_scan_step(x[:, 0], ssm, x[:, 0], A, B[:, 0], B[:, 0])
    for t in (y, o):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            t.sum().backward()
    with torch.inference_mode():      # no versions there: the same numbers
        c2, s2 = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
        S.causal_conv_step(x[:, 0], c2, w)
        S.selective_scan_step(x[:, 0], s2, x[:, 0], A, B[:, 0], B[:, 0])
        assert torch.equal(c2, conv) and torch.equal(s2, ssm)


def test_the_stream_written_in_place_is_refused(S):
    x, r = dev(Draw(4)(3, 16), True), dev(Draw(5)(3, 16))
    y, s = S.add_rms_norm(x, torch.ones(16, device="cuda"), r)
    with torch.no_grad():
        s += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_the_same_tensor_twice(S):
    """Gradients of a tensor in several places are the sums of the places' gradients (fp32: a rounding an addition)."""
    d = Draw(6)
    x, w, A, B = dev(d(2, 40, 16), True), dev(1 + d(16)), -dev(d(16, 8).abs()), dev(d(2, 40, 8), True)
    dy = dev(d(2, 40, 16))
    apart = lambda t, n: [t.detach().clone().requires_grad_() for _ in range(n)]   # noqa: E731

    def same(got, parts):
        terms = torch.stack([p.double() for p in parts])
        P.close(got, terms.sum(0), terms.abs().sum(0), len(parts))

    y, s = S.add_rms_norm(x, w, x)
    a = apart(x, 2)
    y2, s2 = S.add_rms_norm(a[0], w, a[1])
    assert torch.equal(y, y2) and torch.equal(s, s2)
    same(*torch.autograd.grad([y, s], x, [dy, dy]), torch.autograd.grad([y2, s2], a, [dy, dy]))
    o, _ = S.selective_scan(x, x, A, B, B, z=x)
    a, b = apart(x, 3), apart(B, 2)
    o2, _ = S.selective_scan(a[0], a[1], A, b[0], b[1], z=a[2])
    assert torch.equal(o, o2)
    gx, gB = torch.autograd.grad(o, [x, B], dy)
    g = torch.autograd.grad(o2, a + b, dy)
    same(gx, g[:3])
    same(gB, g[3:])


def test_gradients_of_the_last_state_alone_and_of_the_output_alone(S):
    d = Draw(7)
    v = {k: dev(t, k != "starts") for k, t in scan_inputs(d, 2, 45, 24, 16, 1, BF).items()}
    w = dev(d(24, 3), True)
    leaves = [t for k, t in v.items() if k != "starts"]
    dl, dy = dev(d(2, 24, 16)), dev(d(2, 45, 24, dtype=BF))
    o, last = run_scan(S, v)
    for outs, gs, full in (([last], [dl], [torch.zeros_like(o), dl]), ([o], [dy], [dy, torch.zeros_like(last)])):
        got = torch.autograd.grad(outs, leaves, gs, retain_graph=True, materialize_grads=True)
        want = torch.autograd.grad([o, last], leaves, full, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, last = S.causal_conv(v["u"], w, starts=v["starts"])
    dl = dev(d(2, 2, 24, dtype=BF))
    for outs, gs, full in (([last], [dl], [torch.zeros_like(y), dl]), ([y], [dy], [dy, torch.zeros_like(last)])):
        got = torch.autograd.grad(outs, [v["u"], w], gs, retain_graph=True)
        want = torch.autograd.grad([y, last], [v["u"], w], full, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------------- views
def test_broadcast_views_and_their_gradients(S):
    """Rows, batches and gradients that are one row or one batch many times over, against copies of them."""
    d = Draw(8)
    one, w, A, B = d(1, 37, 32), dev(d(32, 4)), -dev(d(32, 16).abs()), d(1, 37, 16)
    dy = dev(d(1, 1, 32)).expand(3, 37, 32)

    def ops(x, B, dy):
        x, B = x.requires_grad_(), B.requires_grad_()
        y, s = S.add_rms_norm(x, w[:, 0], x)
        c, _ = S.causal_conv(x, w, activation="silu")
        o, last = S.selective_scan(x, x, A, B, B)
        with torch.no_grad():
            q = S.quantize_rows(x)
            p = S.matmul_i8(*q, q[0][0, :5], q[1][0, :5])
        return [y, s, c, o, last, p] + [g for t in (y, s, c, o) for g in torch.autograd.grad(t, x, dy, retain_graph=True)] + \
            list(torch.autograd.grad(o, B, dy))

    got = ops(dev(one).expand(3, 37, 32).detach(), dev(B).expand(3, 37, 16).detach(), dy)
    want = ops(dev(one.repeat(3, 1, 1)), dev(B.repeat(3, 1, 1)), dy.contiguous())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_views_that_stand_for_their_negative(S):
    """torch marks such views and leaves the memory as it is."""
    d = Draw(9)
    x, w, A, B, st = dev(d(2, 9, 16)), dev(d(16, 4)), dev(d(16, 4).abs()), dev(d(2, 9, 4)), dev(d(2, 3, 16))
    h = dev(d(2, 16, 4))

    def ops(neg):
        x_, w_, A_, B_, st_, h_ = (neg(t.clone().requires_grad_()) for t in (x, w, A, B, st, h))
        y, _ = S.add_rms_norm(x_, w_[:, 0], x_)
        c, cl = S.causal_conv(x_, w_, w_[:, 0], state=st_)
        o, last = S.selective_scan(x_, x_, A_, B_, B_, state=h_)
        back = torch.autograd.grad([y, c, o], [x_, w_, A_, B_], [neg(x), neg(x), neg(x)])
        with torch.no_grad():
            q, s = S.quantize_rows(x_)
            p = S.matmul_i8(neg(q), s, neg(q[0]), neg(s[0]))
        return [y, c, cl, o, last, q, s, p, *back]

    for a, b in zip(ops(torch._neg_view), ops(torch.neg)):
        assert torch.equal(a, b)
    with torch.no_grad(), pytest.raises(ValueError, match="contiguous"):
        S.causal_conv_step(x[:, 0], torch._neg_view(st), w)


# ---------------------------------------------------------------------------------- odd rows
@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("rows,dim", [(5, 2), (70, 4), (3, 7), (300, 9), (33, 16), (5, 63), (40, 65), (9, 100), (130, 129), (2, 513),
                                      (3, 1025), (2, 4095), (2, 8191), (2, 16401)])
def test_rows_of_any_length(S, dtype, rows, dim):
    """Rows by 8, 16, 32 and 64 lanes, a workgroup and in parts; whole packs of a row and not."""
    T.test_norm_and_gradient(S, dtype, rows, dim)
    T.test_norm_in_8_bits(S, dtype, rows, dim)


@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("dim", [8, 24, 61, 512, 2050])
def test_rows_that_begin_anywhere(S, dtype, dim):
    """Columns cut out of wider tensors, from an odd one on, against copies: the same values, each written once or the same."""
    d = Draw(dim)
    wide_rows = [dev(d(37, dim + 5, dtype=dtype)) for _ in range(4)]
    w = dev(1 + d(dim + 1))

    def ops(x, r, dy, ds, w):
        x, r, w = (t.detach().requires_grad_() for t in (x, r, w))
        y, s = S.add_rms_norm(x, w, r)
        back = torch.autograd.grad([y, s], [x, r, w], [dy, ds])
        with torch.no_grad():
            return [y, s, *back, *S.add_rms_norm_q8(x, w, r), *S.quantize_rows(x)]

    got = ops(*[t[:, 3:3 + dim] for t in wide_rows], w[1:])
    want = ops(*[t[:, 3:3 + dim].contiguous() for t in wide_rows], w[1:].clone())
    for a, b in zip(got, want):       # (the sums of two variants: a few roundings, so a step of the output's type)
        step = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10, torch.int8: 0}[a.dtype]
        a, b = a.double(), b.double()
        assert ((a - b).abs() <= step * b.abs().clamp_min(b.abs().mean()) + (step == 0)).all()
    for t, u in zip(wide_rows, [dev(v) for v in (lambda d: [d(37, dim + 5, dtype=dtype) for _ in range(4)])(Draw(dim))]):
        assert torch.equal(t, u)      # what is around them is as it was


# ---------------------------------------------------------------------------------- products
@pytest.mark.parametrize("M,N", [(1, 40), (19, 33), (40, 20), (64, 17), (70, 65), (300, 257), (1700, 1500), (3600, 3600)])
def test_products_of_rows_that_begin_anywhere(S, M, N):
    """Every alignment of both operands and ends of rows of every length, each variant; the sum is exact."""
    g = torch.Generator().manual_seed(M * N)
    q, w = (torch.randint(-128, 128, (n, 340), generator=g, dtype=torch.int8).cuda() for n in (M, N))
    one, ones = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    for K, i, j in [(1, 0, 3), (5, 1, 1), (15, 2, 0), (16, 3, 2), (17, 0, 1), (63, 1, 2), (64, 16, 0), (65, 0, 0), (79, 3, 3), (127, 2, 1),
                    (128, 0, 16), (130, 1, 0), (191, 0, 2), (192, 7, 9), (257, 0, 0), (300, 5, 4), (321, 1, 3)]:
        a, b = q[:, i:i + K], w[:, j:j + K]
        assert torch.equal(S.matmul_i8(a, one, b, ones).double(), a.double() @ b.double().t()), (K, i, j)
        if M * N < 10 ** 6:    # rows a multiple of 16 apart, as quantize_rows leaves them
            rows = (lambda t: torch.zeros(t.shape[0], (K + 15) // 16 * 16 + 16, dtype=torch.int8, device="cuda")[:, :K].copy_(t))
            assert torch.equal(S.matmul_i8(rows(a), one, rows(b), ones).double(), a.double() @ b.double().t()), K


# ---------------------------------------------------------------------------------- scans
@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("B,L,D,N,G", [(1, 48, 8, 16, 1), (2, 50, 40, 16, 1), (1, 97, 10, 4, 1), (2, 300, 24, 3, 2), (1, 130, 66, 64, 2),
                                       (3, 161, 7, 8, 1), (1, 900, 5, 32, 1)])
def test_scans_cut_in_short_chunks(S, dtype, B, L, D, N, G):
    T.test_scan_and_gradient(S, dtype, B, L, D, N, G)


@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("B,L,D,N,G", [(2101, 3, 8, 16, 1), (1100, 18, 6, 4, 2), (700, 1, 250, 16, 1), (2300, 8, 5, 7, 1), (4099, 2, 9, 2, 1),
                                       (1030, 16, 20, 40, 2)])
def test_scans_of_many_sequences(S, dtype, B, L, D, N, G):
    """More than the chip holds at once: a workgroup takes several."""
    T.test_scan_and_gradient(S, dtype, B, L, D, N, G)


@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("D,N", [(64, 16), (37, 16), (70, 6), (130, 5)])
def test_scans_of_channels_that_begin_anywhere(S, dtype, D, N):
    """u, delta, z, B, C cut out of wider tensors, from an odd column on, against copies of them."""
    d = Draw(D * N)
    one = [dev(d(2, 75, D + 4, dtype=dtype)) for _ in range(4)]
    two = [dev(d(2, 75, N + 3, dtype=dtype)) for _ in range(2)]
    A = -dev(d(D, N).abs())

    def ops(u, delta, z, dy, B, C):
        v = [t.detach().requires_grad_() for t in (u, delta, z, B, C)]
        o, last = S.selective_scan(v[0], v[1], A, v[3], v[4], z=v[2])
        return [o, last, *torch.autograd.grad(o, v, dy)]

    cut = [t[..., 3:3 + D] for t in one] + [t[..., 1:1 + N] for t in two]
    for a, b in zip(ops(*cut), ops(*[t.contiguous() for t in cut])):
        near(a, b, 1)


# ---------------------------------------------------------------------------------- values
@pytest.mark.parametrize("dim,at", [(64, 5), (61, 58), (5, 0), (1003, 999), (20001, 19997)])
def test_rows_with_infinity(S, dim, at):
    x = torch.randn(4, dim, device="cuda")
    x[1, at], x[2, dim // 2], x[3] = float("inf"), float("nan"), 0
    y, _ = S.add_rms_norm(x, torch.ones(dim, device="cuda"))
    assert torch.isfinite(y[0]).all() and torch.isnan(y[2]).all() and not y[3].any()
    assert torch.isnan(y[1, at]) and not y[1, torch.arange(dim) != at].any()
    q, s, _ = S.add_rms_norm_q8(x, torch.ones(dim, device="cuda"))
    assert torch.isnan(s[1:3]).all() and s[3] == 0 and not q[1:].any()


def test_a_growing_state_that_starts_at_zero_in_a_cut_sequence(S):
    """A > 0 over many chunks: the chunks' factors outgrow fp32 (exp(2 * 128)) while the state is zero."""
    d = Draw(10)
    L = 4096
    u, B = d(1, L, 16), d(1, L, 1, 8)
    u[:, :2048] = 0
    delta = torch.where(torch.arange(L) < 2048, 0.5, -20.0)[None, :, None].expand(1, L, 16).contiguous()
    v = dict(u=u, delta=delta, A=torch.full((16, 8), 2.0), B=B, C=d(1, L, 1, 8), D=None, z=None, bias=None, starts=None, state=None)
    out, last = run_scan(S, {k: dev(t) for k, t in v.items()})
    ro, rl, eo, el = plain_scan(v)
    assert not out[:, :2048].any() and torch.isfinite(out).all()
    P.close(out, ro, eo, 1, "out")
    P.close(last, rl, el, 1, "last")


# ---------------------------------------------------------------------------------- sizes
def test_sizes_past_what_is_held_in_32_bits_are_refused(S):
    n = 2 ** 32 + 16      # 16, to who keeps 32 bits of it
    one = torch.ones(1, device="cuda", dtype=BF)
    x, w = one.expand(1, n), one.expand(n)
    for call in (lambda: S.add_rms_norm(x, w), lambda: S.add_rms_norm_q8(x, w), lambda: S.quantize_rows(x),
                 lambda: S.causal_conv(x[None], one.expand(n, 4)), lambda: S.causal_conv_step(x, one.expand(1, 3, n), one.expand(n, 4)),
                 lambda: S.selective_scan(x[None], x[None], one.expand(n, 4), one.expand(1, 1, 4), one.expand(1, 1, 4)),
                 lambda: S.selective_scan_step(x, one.float().expand(1, n, 4), x, one.expand(n, 4), one.expand(1, 4), one.expand(1, 4)),
                 lambda: S.matmul_i8(one.to(torch.int8).expand(1, n), one, one.to(torch.int8).expand(1, n), one)):
        with pytest.raises(ValueError):
            call()


@pytest.fixture(scope="module")
def tall():
    """2^20 + 3 rows of 4096: more elements than 32 bits count."""
    if torch.cuda.get_device_properties(0).total_memory < 200e9:
        pytest.skip("needs a device with more than 200 GB")
    x = torch.empty(2 ** 20 + 3, 4096, dtype=BF, device="cuda")
    torch.manual_seed(0)
    for part in x.split(2 ** 18):
        part.normal_()
    yield x
    del x
    torch.cuda.empty_cache()


END = 70     # rows compared: a run of their own gives them too


def test_offsets_past_32_bits_norm_and_product(S, tall):
    w = 1 + 0.1 * torch.randn(4096, device="cuda")
    x = tall.requires_grad_()
    y, _ = S.add_rms_norm(x, w)
    gx, = torch.autograd.grad(y, x, tall.detach())
    x2 = tall[-END:].detach().clone().requires_grad_()
    y2, _ = S.add_rms_norm(x2, w)
    g2, = torch.autograd.grad(y2, x2, x2.detach())
    assert torch.equal(y[-END:], y2) and torch.equal(gx[-END:], g2)
    tall.requires_grad_(False)
    del x, y, gx
    q, s = S.quantize_rows(tall)
    q2, s2 = S.quantize_rows(tall[-END:])
    assert torch.equal(q[-END:], q2) and torch.equal(s[-END:], s2)
    wq, ws = S.quantize_rows(torch.randn(4096, 64, device="cuda"))
    for k in (16, 4096):      # long rows of q; then many columns of the output
        a, b = (q, wq[:16].repeat(1, 64)) if k == 4096 else (q[:, :64], wq)
        o = S.matmul_i8(a, s, b, ws[:b.shape[0]], out_dtype=BF)
        assert torch.equal(o[-END:], S.matmul_i8(a[-END:].contiguous(), s2, b, ws[:b.shape[0]], out_dtype=BF))
        del o


def test_offsets_past_32_bits_convolution(S, tall):
    w = torch.randn(4096, 4, device="cuda")
    x = tall[None].requires_grad_()
    y, last = S.causal_conv(x, w, activation="silu")
    gx, = torch.autograd.grad(y, x, x.detach())
    x2 = tall[None, -END:].detach().clone().requires_grad_()
    y2, last2 = S.causal_conv(x2, w, activation="silu", state=tall[None, -END - 3:-END].detach())
    g2, = torch.autograd.grad(y2, x2, x2.detach())
    assert torch.equal(y[:, -END:], y2) and torch.equal(gx[:, -END:], g2) and torch.equal(last, last2)


def test_offsets_past_32_bits_scan(S, tall):
    """The end is a sequence of its own (a start); at most one step of bf16 off, the two runs' tiles lying differently."""
    L = tall.shape[0]
    A, B = -torch.rand(4096, 16, device="cuda") - 0.1, torch.randn(1, L, 16, device="cuda", dtype=BF)
    starts = torch.zeros(1, L, dtype=torch.bool, device="cuda")
    starts[0, -END] = True

    def run(x, B, starts):
        x, B = x.requires_grad_(), B.requires_grad_()
        y, last = S.selective_scan(x, x, A, B, B, z=x, starts=starts)
        return [y[:, -END:], last] + [g[:, -END:] for g in torch.autograd.grad(y, [x, B], x.detach())]

    got = run(tall[None].detach(), B, starts)
    want = run(tall[None, -END:].detach().clone(), B[:, -END:].detach().clone(), starts[:, -END:].contiguous())
    for a, b in zip(got, want):
        near(a, b, 4)     # (x's gradient is the sum of three, each rounded to bf16 and each maybe a step off)


def test_offsets_past_32_bits_steps(S):
    if torch.cuda.get_device_properties(0).total_memory < 200e9:
        pytest.skip("needs a device with more than 200 GB")
    n, d = 2 ** 20 + 5, 2048
    torch.manual_seed(1)
    x, w = torch.randn(n, d, device="cuda", dtype=BF), torch.randn(d, 4, device="cuda")
    conv = torch.zeros(n, 3, d, device="cuda", dtype=BF)
    conv[-END:].normal_()
    c2 = conv[-END:].clone()
    assert conv.numel() > 2 ** 32
    y, y2 = S.causal_conv_step(x, conv, w), S.causal_conv_step(x[-END:], c2, w)
    assert torch.equal(y[-END:], y2) and torch.equal(conv[-END:], c2)
    del conv, y
    torch.cuda.empty_cache()
    n = 2 ** 17 + 5
    ssm = torch.zeros(n, d, 16, device="cuda")
    ssm[-END:].normal_()
    s2 = ssm[-END:].clone()
    assert ssm.numel() > 2 ** 32
    A, B = -torch.rand(d, 16, device="cuda"), torch.randn(n, 16, device="cuda", dtype=BF)
    u = x[:n]
    y = S.selective_scan_step(u, ssm, u, A, B, B, z=u)
    y2 = S.selective_scan_step(u[-END:], s2, u[-END:], A, B[-END:], B[-END:], z=u[-END:])
    near(y[-END:], y2, 1)
    near(ssm[-END:], s2, 1)
    del ssm, y
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------- graphs
def test_captured_steps_carry_their_states(S):
    """Two captured graphs of a step, each with states of its own, replayed in turn against eager steps."""
    d = Draw(11)
    w, A = dev(d(32, 4)), -dev(d(32, 16).abs())
    wq = None

    def step(x, conv, ssm, reset):
        nonlocal wq
        u = S.causal_conv_step(x, conv, w, activation="silu", reset=reset)
        q, s, _ = S.add_rms_norm_q8(u, w[:, 0], x)
        p = S.matmul_i8(q, s, *wq)
        return S.selective_scan_step(u, ssm, p[:, :32], A, p[:, 32:48], p[:, 48:], z=x, reset=reset)

    def new():
        return [dev(d(70, 32)), torch.zeros(70, 3, 32, device="cuda"), torch.zeros(70, 32, 16, device="cuda"),
                torch.zeros(70, dtype=torch.uint8, device="cuda")]

    wq = S.quantize_rows(dev(d(64, 32)))
    sets, graphs = [new(), new()], []
    mirror = [[t.clone() for t in s] for s in sets]
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*[t.clone() for t in s])
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.append(step(*s))
        graphs.append(g)
    for k in range(6):
        for s, m in zip(sets, mirror):
            x, r = dev(d(70, 32)), dev(d.starts(70))
            for to in (s, m):
                to[0].copy_(x)
                to[3].copy_(r)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, m in zip(sets, mirror):
            want = step(*m)
            assert torch.equal(s[4], want) and torch.equal(s[1], m[1]) and torch.equal(s[2], m[2]), k


# ---------------------------------------------------------------------------------- 8 bits next to halves
def halves(rows, dim, dtype, g):
    """Rows whose values lie on both sides of the halves between two steps of 8 bits, up to two steps of fp32 away."""
    top = (torch.rand(rows, 1, generator=g) * 3 + 0.5).to(dtype).float()
    x = ((torch.randint(0, 127, (rows, dim), generator=g) + 0.5) * (top / 127)).to(dtype)
    if dtype == torch.float32:
        x = x.view(torch.int32).add(torch.randint(-2, 3, (rows, dim), generator=g, dtype=torch.int32)).view(torch.float32)
    x = x * torch.where(torch.rand(rows, dim, generator=g) < 0.5, -1, 1).to(dtype)
    x[:, dim // 2] = top[:, 0].to(dtype)
    return x


@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("dim", [3, 40, 64, 333, 1024, 2047, 9000, 20001])
def test_8_bits_are_the_rounded_quotient(S, dtype, dim):
    """q is the fp32 quotient by the scale rounded to nearest even, next to halves too (the product with 1 / scale is not)."""
    x = halves(max(300, 200000 // dim), dim, dtype, torch.Generator().manual_seed(dim))
    q, scale = S.quantize_rows(dev(x))
    top = x.float().abs().amax(1) / 127
    assert torch.equal(scale.cpu(), top)
    assert torch.equal(q.cpu(), torch.round(x.float() / top[:, None]).to(torch.int8))


@pytest.mark.parametrize("rows,dim", [(8192, 2048), (60000, 256), (900, 20001)])
def test_8_bits_of_the_norm_are_the_rounded_quotient(S, rows, dim):
    """fp32: y as it is before 8 bits is the norm's own output (the same arithmetic)."""
    x, w = torch.randn(rows, dim, device="cuda"), 1 + 0.1 * torch.randn(dim, device="cuda")
    with torch.no_grad():
        y, _ = S.add_rms_norm(x, w)
        q, scale, _ = S.add_rms_norm_q8(x, w)
    y, scale = y.cpu(), scale.cpu()
    assert torch.equal(scale, y.abs().amax(1) / 127)
    assert torch.equal(q.cpu(), torch.round(y / scale[:, None]).to(torch.int8))


@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=T.ids)
def test_8_bits_of_small_rows(S, dtype):
    """Down to the least normal scale, and 0 below it.  A power of two changes the scale and nothing else, but for fp32
    at 2^-118: scales there begin at 2^-126, and half of such a one is below the normal numbers, where x itself is rounded
    (spacing 2^-149).  So the rounded quotient of what x is decides."""
    x = halves(700, 333, dtype, torch.Generator().manual_seed(1))
    _, scale = S.quantize_rows(x.cuda())
    for e in (-50, -70, -100, -118):
        x2 = x * 2.0 ** e
        q2, s2 = S.quantize_rows(x2.cuda())
        assert torch.equal(s2, scale * 2.0 ** e), e
        assert torch.equal(q2.cpu(), torch.round(x2.float() / s2.cpu()[:, None]).to(torch.int8)), e
    q2, s2 = S.quantize_rows(x.cuda() * 2.0 ** -122)
    assert not q2.any() and not s2.any()


# ---------------------------------------------------------------------------------- starts of growing states
@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("L,N", [(40, 4), (40, 16), (900, 8)])
def test_a_start_whose_decay_outgrows_fp32(S, dtype, L, N):
    """exp(dt A) = exp(12 * 10) at the starts: its place is taken by 0, not by a product with a state of 0."""
    d = Draw(L + N)
    v = scan_inputs(d, 2, L, 24, N, 1, dtype)
    v["A"], v["bias"] = torch.full((24, N), 10.0), None
    v["starts"] = d.starts(2, L, p=0.05)
    v["starts"][:, 0] = 1
    v["delta"] = torch.where(v["starts"][..., None] != 0, 12.0, -9.0).expand(2, L, 24).to(dtype).contiguous()
    T.check_scan(S, v, d, dtype)
    for t in (0, L // 2):      # one token at a time, each the start of a sequence
        g = {k: dev(x) for k, x in v.items()}
        h = g["state"].clone()
        y = S.selective_scan_step(g["u"][:, t], h, torch.full_like(g["u"][:, t], 12.0), g["A"], g["B"][:, t], g["C"][:, t],
                                  reset=torch.ones(2, dtype=torch.bool, device="cuda"))
        one = {k: x if k in ("A", "state") else None if x is None or k in ("D", "z") else x[:, t:t + 1] for k, x in v.items()}
        one["delta"], one["starts"] = torch.full_like(one["u"], 12.0), torch.ones(2, 1, dtype=torch.uint8)
        ro, rl, eo, el = plain_scan(one)
        P.close(y[:, None], ro, eo, 1, "out")
        P.close(h, rl, el, 1, "state")


# ---------------------------------------------------------------------------------- forward mode
def test_tangents_are_refused_back_as_well(S):
    import torch.autograd.forward_ad as fwad
    x, w, A, B = dev(Draw(1)(2, 9, 16), True), torch.ones(16, 4, device="cuda"), -torch.ones(16, 4, device="cuda"), dev(Draw(2)(2, 9, 4))
    outs = [S.add_rms_norm(x, w[:, 0])[0], S.add_rms_norm(x, w[:, 0], x)[1], S.causal_conv(x, w)[0], S.selective_scan(x, x, A, B, B)[0]]
    with fwad.dual_level():
        for y in outs:
            dy = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(y, x, dy)
        d = fwad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: S.add_rms_norm(d, w[:, 0]), lambda: S.causal_conv(d, w), lambda: S.selective_scan(d, x, A, B, B)):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call()
        with torch.inference_mode():      # where torch itself goes without tangents
            assert torch.equal(S.add_rms_norm(d, w[:, 0])[0], S.add_rms_norm(x, w[:, 0])[0])


# ---------------------------------------------------------------------------------- sizes of one launch
def test_a_product_of_more_tokens_than_small_tiles_would_serve(S):
    """2^29 + 5 tokens: past 2^23 tiles of 64 x 64, which nothing uses at this size."""
    if torch.cuda.get_device_properties(0).total_memory < 200e9:
        pytest.skip("needs a device with more than 200 GB")
    M, K = 2 ** 29 + 5, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device="cuda")
    w = torch.randint(-128, 128, (3, K), generator=g, dtype=torch.int8, device="cuda")
    out = S.matmul_i8(q, torch.ones(M, device="cuda"), w, torch.ones(3, device="cuda"))
    for part in (slice(0, END), slice(2 ** 28 - 7, 2 ** 28 + 300), slice(M - END, M)):
        assert torch.equal(out[part].double(), q[part].double() @ w.double().t().contiguous())
    del q, out
    torch.cuda.empty_cache()


def test_a_scan_of_more_states_than_a_chain_would_serve(S):
    """2^17 + 5 sequences of one token, 2048 channels, 16 states: 2^30 lanes of 4 states; no chunks, so nothing is chained."""
    if torch.cuda.get_device_properties(0).total_memory < 200e9:
        pytest.skip("needs a device with more than 200 GB")
    n, d = 2 ** 17 + 5, 2048
    torch.manual_seed(2)
    x, B, A = torch.randn(n, 1, d, device="cuda", dtype=BF), torch.randn(n, 1, 16, device="cuda", dtype=BF), -torch.rand(d, 16, device="cuda")

    def run(x, B):
        x, B = x.detach().requires_grad_(), B.detach().requires_grad_()
        y, last = S.selective_scan(x, x, A, B, B, z=x)
        return [t[-END:].clone() for t in (y.detach(), last.detach(), *torch.autograd.grad(y, [x, B], x.detach()))]

    got = run(x, B)
    torch.cuda.empty_cache()
    for a, b in zip(got, run(x[-END:], B[-END:])):      # (the same kernels: a sequence's arithmetic is its own)
        assert torch.equal(a, b)
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------- the product's largest tiles
@pytest.mark.parametrize("dtype", T.TYPES, ids=T.ids)
@pytest.mark.parametrize("M,N", [(3600, 3600), (6001, 2050), (2049, 5384)])
@pytest.mark.parametrize("K", [16, 64, 80, 128, 192, 208, 256, 320, 1040])
def test_products_of_large_tiles_over_many_stages(S, dtype, M, N, K):
    """Rows on 16-byte boundaries, 192 tiles of 256 x 256 and more; every element, whole and partial last stages.  Roundings:
    the sum's in fp32, two products, the bias's addition."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    q, w = (torch.randint(-128, 128, (n, K), generator=g, dtype=torch.int8, device="cuda") for n in (M, N))
    s, ws, b = (torch.rand(n, generator=g, device="cuda") + 0.01 for n in (M, N, N))
    if dtype == torch.float16:
        s = s * 2.0 ** -12      # (sums of 16 million would overflow half precision)
    out = S.matmul_i8(q, s, w, ws, bias=b, out_dtype=dtype).double()
    scaled = q.double() @ w.double().t().contiguous() * s.double()[:, None] * ws.double()
    slack = 4 * P.E32 * (scaled.abs() + b.double())
    ref = scaled + b.double()
    assert ((out - ref).abs() <= slack + P.STEP[dtype] * (ref.abs() + slack) + P.TINY[dtype]).all()


# ---------------------------------------------------------------------------------- a step's inputs in its state
def test_steps_whose_inputs_lie_in_their_state(S):
    """Views of the state that a step advances in place, as its inputs: what they held before the call."""
    d = Draw(12)
    n, dim, N = 300, 520, 16
    state, w = dev(d(n, 3, dim)), dev(d(dim, 4))
    flat = state.view(n, -1)
    for x in (flat[:, 7:7 + dim], flat[:, 1030:1030 + dim], state[:, 2], flat[:1, :dim].expand(n, dim)):
        want_state, want_x = state.clone(), x.clone()
        held = state.clone()
        want = S.causal_conv_step(want_x, want_state, w)
        assert torch.equal(S.causal_conv_step(x, state, w), want) and torch.equal(state, want_state)
        state.copy_(held)
    h, A, B, u = dev(d(n, dim, N)), -dev(d(dim, N).abs()), dev(d(n, N)), dev(d(n, dim))
    flat = h.view(n, -1)
    for v in (dict(u=flat[:, 100:100 + dim]), dict(B=h[:, 5], C=h[:, dim - 1]), dict(A=h[n - 1]), dict(delta=flat[:, -dim:], z=flat[:, :dim]),
              dict(D=flat[3, :dim], B=h[:1, 0].expand(n, N))):
        held = h.clone()
        call = lambda h, v: S.selective_scan_step(v.get("u", u), h, v.get("delta", u), v.get("A", A), v.get("B", B), v.get("C", B),   # noqa: E731
                                                  D=v.get("D"), z=v.get("z"))
        want_h = h.clone()
        want = call(want_h, {k: t.clone() for k, t in v.items()})
        assert torch.equal(call(h, v), want) and torch.equal(h, want_h), v.keys()
        h.copy_(held)
