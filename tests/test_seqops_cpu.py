"""Sequence operators on the CPU: refusals of the Python and C entry points (checked before any HIP
call), the ctypes mirrors of their descriptors, and the test formulas of tests/seq_plain.py against
differences."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

import seq_plain as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------------------------- the test's own formulas
def rnd(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("L,W", [(1, 4), (2, 4), (5, 3), (7, 2)])
def test_plain_conv_gradient_against_differences(silu, L, W):
    g = torch.Generator().manual_seed(L * 10 + W)
    x, w, b, st = rnd(g, 2, L, 3), rnd(g, 3, W), rnd(g, 3), rnd(g, 2, W - 1, 3)
    starts = (torch.rand(2, L, generator=g) < 0.3).to(torch.uint8)
    dy, dl = rnd(g, 2, L, 3), rnd(g, 2, W - 1, 3)
    _, _, _, grads, _ = P.conv(x, w, b, silu, starts, st, dy, dl)

    def loss(v):
        y, last, _ = P.conv(v["x"], v["w"], v["b"], silu, starts, v["state"])
        return (y * dy).sum() + (last * dl).sum()
    differences(loss, dict(x=x, w=w, b=b, state=st), grads, g)


@pytest.mark.parametrize("L,G,gate", [(1, 1, True), (6, 2, True), (9, 1, False)])
def test_plain_scan_gradient_against_differences(L, G, gate):
    g = torch.Generator().manual_seed(L)
    d, N = 4, 3
    v = dict(u=rnd(g, 2, L, d), delta=rnd(g, 2, L, d), A=-rnd(g, d, N).abs(), B=rnd(g, 2, L, G, N), C=rnd(g, 2, L, G, N),
             D=rnd(g, d), z=rnd(g, 2, L, d) if gate else None, bias=rnd(g, d), state=rnd(g, 2, d, N))
    starts = (torch.rand(2, L, generator=g) < 0.3).to(torch.uint8)
    dout, dl = rnd(g, 2, L, d), rnd(g, 2, d, N)
    run = lambda v, **k: P.scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], starts, v["state"], **k)  # noqa: E731
    grads = run(v, dout=dout, dlast=dl)[4]

    def loss(v):
        out, h, _, _ = run(v)
        return (out * dout).sum() + (h * dl).sum()
    differences(loss, v, grads, g)


def test_plain_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    s, w, dy, ds = rnd(g, 3, 5), rnd(g, 5), rnd(g, 3, 5), rnd(g, 3, 5)
    dx, _, dw, _ = P.norm_grad(s, w, 1e-6, dy, ds)
    differences(lambda v: (P.norm(v["s"], v["w"], 1e-6)[0] * dy).sum() + (v["s"] * ds).sum(), dict(s=s, w=w), dict(s=dx, w=dw), g)


def differences(loss, v, grads, g):
    """Central differences along a random direction of each input: off by h^2 of third derivatives (1e-10 here) and
    2^-53 / h of the loss (1e-10)."""
    for name, t in v.items():
        if t is None:
            continue
        way = rnd(g, *t.shape)
        h = 1e-5
        got = (loss({**v, name: t + h * way}) - loss({**v, name: t - h * way})) / (2 * h)
        want = (grads[name] * way).sum()
        assert abs(got - want) < 1e-6 * (1 + abs(want)), (name, float(got), float(want))


# ---------------------------------------------------------------------------------- descriptors
@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_descriptor_layouts_match_c(tmp_path):
    from pnp_amd import _lib
    structs = {"pnp_norm_desc": _lib.PnpNormDesc, "pnp_norm_bwd_desc": _lib.PnpNormBwdDesc, "pnp_i8_desc": _lib.PnpI8Desc,
               "pnp_conv_desc": _lib.PnpConvDesc, "pnp_conv_bwd_desc": _lib.PnpConvBwdDesc, "pnp_scan_desc": _lib.PnpScanDesc,
               "pnp_scan_bwd_desc": _lib.PnpScanBwdDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "pnp.h"', "int main(void) {"]
    for c, cls in structs.items():
        lines.append(f'  printf("{c} sizeof %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["  return 0;\n}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict()
    for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"):
        if ln:
            s, f, n = ln.split()
            got[s, f] = int(n)
    for c, cls in structs.items():
        assert got[c, "sizeof"] == C.sizeof(cls), c
        for f, _ in cls._fields_:
            assert got[c, f] == getattr(cls, f).offset, (c, f)


# ---------------------------------------------------------------------------------- C refusals
def _norm():
    from pnp_amd import _lib
    d = _lib.PnpNormDesc()
    d.rows, d.dim, d.type, d.res_type, d.eps = 4, 8, 1, 1, 1e-6
    d.x, d.x_stride, d.y = 4096, 8, 8192
    return d


def _i8():
    from pnp_amd import _lib
    d = _lib.PnpI8Desc()
    d.M, d.N, d.K, d.out_type, d.q_stride, d.wq_stride = 4, 8, 16, 0, 16, 16
    d.q = d.wq = d.scale = d.wscale = d.out = 4096
    return d


def _conv():
    from pnp_amd import _lib
    d = _lib.PnpConvDesc()
    d.B, d.L, d.dim, d.width, d.type = 2, 3, 8, 4, 0
    d.x = d.weight = d.y = 4096
    return d


def _scan():
    from pnp_amd import _lib
    d = _lib.PnpScanDesc()
    d.B, d.L, d.dim, d.N, d.groups, d.type = 2, 1, 8, 16, 1, 0
    d.u = d.delta = d.Bm = d.Cm = d.A = d.out = d.last_state = 4096
    return d


@pytest.mark.parametrize("make,fn,field,value", [
    (_norm, "pnp_rms_norm", "dim", 0), (_norm, "pnp_rms_norm", "rows", -1), (_norm, "pnp_rms_norm", "type", 3),
    (_norm, "pnp_rms_norm", "res_type", 2), (_norm, "pnp_rms_norm", "x", None), (_norm, "pnp_rms_norm", "y", None),
    (_norm, "pnp_rms_norm", "q", 4096), (_norm, "pnp_rms_norm", "residual", 4096),
    (_i8, "pnp_matmul_i8", "K", 0), (_i8, "pnp_matmul_i8", "K", 131072), (_i8, "pnp_matmul_i8", "N", 0),
    (_i8, "pnp_matmul_i8", "M", -1), (_i8, "pnp_matmul_i8", "q_stride", 15), (_i8, "pnp_matmul_i8", "wscale", None),
    (_i8, "pnp_matmul_i8", "out_type", -1),
    (_conv, "pnp_causal_conv", "width", 5), (_conv, "pnp_causal_conv", "width", 1), (_conv, "pnp_causal_conv", "dim", 0),
    (_conv, "pnp_causal_conv", "L", -1), (_conv, "pnp_causal_conv", "x", None), (_conv, "pnp_causal_conv", "type", 9),
    (_scan, "pnp_selective_scan", "N", 65), (_scan, "pnp_selective_scan", "N", 0), (_scan, "pnp_selective_scan", "groups", 3),
    (_scan, "pnp_selective_scan", "A", None), (_scan, "pnp_selective_scan", "out", None),
    (_scan, "pnp_selective_scan", "B", 1 << 31), (_scan, "pnp_selective_scan_step", "L", 2),
    (_scan, "pnp_selective_scan_step", "last_state", None),
])
def test_c_entry_points_refuse(make, fn, field, value):
    from pnp_amd import _lib
    L = _lib.load()
    d = make()
    setattr(d, field, value)
    assert getattr(L, fn)(C.byref(d), None) == -1
    assert fn.encode() in L.pnp_last_error()
    assert getattr(L, fn)(None, None) == -1


def test_c_gradients_refuse_small_workspaces():
    from pnp_amd import _lib
    L = _lib.load()
    n = _lib.PnpNormBwdDesc()
    n.rows, n.dim, n.type, n.res_type = 100, 64, 0, 0
    n.dy = n.s = n.rstd = n.dx = n.dweight = n.workspace = 4096
    need = L.pnp_rms_norm_bwd_workspace(C.byref(n))
    assert need >= 64
    n.workspace_floats = need - 1
    assert L.pnp_rms_norm_bwd(C.byref(n), None) == -1 and b"workspace" in L.pnp_last_error()
    c = _lib.PnpConvBwdDesc()
    c.f = _conv()
    c.dy = c.dx = c.dweight = c.workspace = 4096
    c.workspace_floats = L.pnp_causal_conv_bwd_workspace(C.byref(c)) - 1
    assert c.workspace_floats >= 8 * 5 - 1
    assert L.pnp_causal_conv_bwd(C.byref(c), None) == -1 and b"workspace" in L.pnp_last_error()
    s = _lib.PnpScanBwdDesc()
    s.f = _scan()
    s.f.ckpt_floats = L.pnp_scan_ckpt_floats(C.byref(s.f))
    s.f.ckpt = 4096
    s.dout = s.du = s.ddelta = s.dB = s.dC = s.dA = s.workspace = 4096
    s.workspace_floats = L.pnp_scan_bwd_workspace(C.byref(s)) - 1
    assert L.pnp_selective_scan_bwd(C.byref(s), None) == -1 and b"workspace" in L.pnp_last_error()
    s.f.ckpt_floats -= 1
    assert L.pnp_selective_scan_bwd(C.byref(s), None) == -1 and b"ckpt" in L.pnp_last_error()
    f = _scan()     # a long sequence of few channels is cut: its workspace is asked for
    f.B, f.L = 1, 100_000
    need = L.pnp_scan_workspace(C.byref(f))
    assert need > 0
    f.workspace, f.workspace_floats = 4096, need - 1
    assert L.pnp_selective_scan(C.byref(f), None) == -1 and b"workspace" in L.pnp_last_error()


def test_c_scan_refuses_strides_and_channels_out_of_range():
    """Offsets within a tile are 32-bit; the gradient's last sums are one launch over dim * (N + 2) columns."""
    from pnp_amd import _lib
    L = _lib.load()
    for field in ("u_tstride", "delta_tstride", "z_tstride", "B_tstride", "C_tstride"):
        for value in ((1 << 24) + 1, -1):
            f = _scan()
            setattr(f, field, value)
            assert L.pnp_selective_scan(C.byref(f), None) == -1 and b"stride" in L.pnp_last_error()
    s = _lib.PnpScanBwdDesc()
    s.f = _scan()
    s.f.B, s.f.L = 1, 1
    s.f.ckpt = s.dout = s.du = s.ddelta = s.dB = s.dC = s.dA = s.workspace = 4096
    s.f.ckpt_floats = s.workspace_floats = 1 << 60
    s.dout_tstride = (1 << 24) + 1
    assert L.pnp_selective_scan_bwd(C.byref(s), None) == -1 and b"stride" in L.pnp_last_error()
    s.dout_tstride = 0
    s.f.dim, s.f.N = 1 << 22, 62
    assert L.pnp_selective_scan_bwd(C.byref(s), None) == -1 and b"too many channels" in L.pnp_last_error()


def test_c_empty_batches_launch_nothing():
    from pnp_amd import _lib
    L = _lib.load()
    for make, fn, field in ((_norm, "pnp_rms_norm", "rows"), (_i8, "pnp_matmul_i8", "M"), (_conv, "pnp_causal_conv", "B"),
                            (_scan, "pnp_selective_scan", "B"), (_scan, "pnp_selective_scan_step", "B")):
        d = make()
        setattr(d, field, 0)
        assert getattr(L, fn)(C.byref(d), None) == 0, fn


# ---------------------------------------------------------------------------------- Python refusals
def test_no_cpu_path():
    from pnp_amd import seqops as S
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    for call in (lambda: S.add_rms_norm(x, w), lambda: S.add_rms_norm_q8(x, w), lambda: S.quantize_rows(x),
                 lambda: S.matmul_i8(torch.zeros(2, 8, dtype=torch.int8), torch.ones(2), torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)),
                 lambda: S.causal_conv(x, torch.ones(8, 4)), lambda: S.causal_conv_step(x[:, 0], x, torch.ones(8, 4)),
                 lambda: S.selective_scan(x, x, -torch.ones(8, 4), x[..., :4], x[..., :4]),
                 lambda: S.selective_scan_step(x[:, 0], torch.zeros(2, 8, 4), x[:, 0], -torch.ones(8, 4), x[:, 0, :4], x[:, 0, :4])):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_serving_calls_refuse_gradients():
    from pnp_amd import seqops as S
    x = torch.zeros(2, 8, requires_grad=True)
    for call in (lambda: S.add_rms_norm_q8(x, torch.ones(8)), lambda: S.quantize_rows(x),
                 lambda: S.causal_conv_step(x, x, torch.ones(8, 4)),
                 lambda: S.selective_scan_step(x, x, x, x, x, x)):
        with pytest.raises(ValueError, match="no gradient"):
            call()


def test_forward_mode_derivatives_are_refused():
    """A tangent is never dropped: the operators have gradients, and no derivative forward."""
    import torch.autograd.forward_ad as fwad
    from pnp_amd import seqops as S
    x, w, A = torch.zeros(2, 3, 8), torch.ones(8, 4), -torch.ones(8, 4)
    B, h, i8 = torch.zeros(2, 3, 4), torch.zeros(2, 8, 4), torch.zeros(2, 8, dtype=torch.int8)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))   # noqa: E731
        for call in (lambda: S.add_rms_norm(dual(x), w[:, 0]), lambda: S.add_rms_norm(x, dual(w[:, 0])),
                     lambda: S.add_rms_norm(x, w[:, 0], dual(x)), lambda: S.causal_conv(dual(x), w), lambda: S.causal_conv(x, dual(w)),
                     lambda: S.causal_conv(x, w, dual(w[:, 0])), lambda: S.causal_conv(x, w, state=dual(x)),
                     lambda: S.selective_scan(dual(x), x, A, B, B), lambda: S.selective_scan(x, dual(x), A, B, B),
                     lambda: S.selective_scan(x, x, dual(A), B, B), lambda: S.selective_scan(x, x, A, dual(B), B),
                     lambda: S.selective_scan(x, x, A, B, dual(B)), lambda: S.selective_scan(x, x, A, B, B, D=dual(w[:, 0])),
                     lambda: S.selective_scan(x, x, A, B, B, z=dual(x)), lambda: S.selective_scan(x, x, A, B, B, delta_bias=dual(w[:, 0])),
                     lambda: S.selective_scan(x, x, A, B, B, state=dual(h)),
                     lambda: S.add_rms_norm_q8(dual(x), w[:, 0]), lambda: S.quantize_rows(dual(x)),
                     lambda: S.matmul_i8(i8, dual(w[:2, 0]), i8, w[:2, 0]), lambda: S.causal_conv_step(x[:, 0], dual(x), w),
                     lambda: S.selective_scan_step(dual(x[:, 0]), h, x[:, 0], A, B[:, 0], B[:, 0]),
                     lambda: S.selective_scan_step(x[:, 0], dual(h), x[:, 0], A, B[:, 0], B[:, 0])):
            for mode in (torch.enable_grad, torch.no_grad):   # (forward mode does not ask for either)
                with mode(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                    call()
        with pytest.raises(ValueError, match="no CPU path"):      # a dual level by itself is nothing to refuse
            S.add_rms_norm(x, w[:, 0])
    with pytest.raises(ValueError, match="no CPU path"):
        S.quantize_rows(x)


def test_c_product_refuses_more_tiles_than_a_launch_holds():
    from pnp_amd import _lib
    L = _lib.load()
    d = _i8()
    d.M, d.N = 1 << 31, 257          # 2^23 * 2 tiles
    assert L.pnp_matmul_i8(C.byref(d), None) == -1 and b"too many tiles" in L.pnp_last_error()
    d.N = 1
    assert L.pnp_matmul_i8(C.byref(d), None) == -1 and b"too many tiles" in L.pnp_last_error()


def test_c_scan_refuses_more_sequences_than_a_launch_holds():
    from pnp_amd import _lib
    L = _lib.load()
    d = _scan()
    for B, dim, N, groups in ((1 << 24, 8, 16, 1), (1 << 23, 16, 16, 2), (1 << 20, 257 * 8, 64, 1), (1 << 20, 16, 1, 16)):
        d.B, d.dim, d.N, d.groups = B, dim, N, groups
        assert L.pnp_selective_scan(C.byref(d), None) == -1 and b"too many sequences" in L.pnp_last_error()


# ---------------------------------------------------------------------------------- build
@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_objects_are_built_anew_where_their_flags_change():
    """The Makefile holds the compiler's flags: objects of others must not be linked."""
    csrc = os.path.join(ROOT, "mujoco-panda-pnp_amd", "csrc")
    plan = subprocess.run(["make", "-n", "-W", "Makefile", "-C", csrc], check=True, capture_output=True, text=True).stdout
    for unit in ("seq_norm.hip", "seq_scan.hip", "tqc_fused.hip", "step.hip", "ik_dls.hip", "resident.cpp", "seq_torch.cpp"):
        assert unit in plan, unit
