"""Operators of a policy with memory on device tensors: the layers of ``pnp_amd.history`` (and of
any other sequence model a user builds beside it), each by hand-written HIP kernels of libpnp.so
(include/pnp.h, csrc/seq_*.hip).

* ``add_rms_norm``            residual addition and root-mean-square norm, with its gradient
* ``add_rms_norm_q8``         the same with an 8-bit output and a scale per row
* ``quantize_rows``           rows in 8 bits with a scale each (tokens, or a weight's output channels)
* ``matmul_i8``               product in 8-bit integers, a scale per token and per output channel
* ``causal_conv``             short causal convolution per channel, with its gradient
* ``causal_conv_step``        its form for one token of each of many sequences
* ``selective_scan``          selective state space scan, with its gradient
* ``selective_scan_step``     its form for one token of each of many sequences

Activations are fp32, bf16 or fp16 (one type within a call); states, statistics and sums are fp32;
weights, biases, ``A`` and ``D`` are taken in any floating type and used in fp32.  Tensors may have any
strides (a last dimension that is not contiguous is copied first); outputs are contiguous.  Launches go
on the tensors' device, on its current stream; nothing synchronises; every call takes its workspace from
torch's allocator, so calls on several streams and in several captured graphs do not share one.  The same
call gives the same bits.  There is no CPU path: a CPU tensor is a ``ValueError``.

Sequences that end inside a batch: ``starts`` [B, L] (uint8 or bool) marks tokens that begin a new
sequence; they and what follows see nothing from before, whatever it holds (infinities and NaN
included).  Sequences of different lengths go padded on the left, with a start at the first real token;
packed sequences go one after the other in a row.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_byref = C.byref   # (C names a tensor in the scan's calls)
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # PNP_F32, PNP_BF16, PNP_F16


# ---------------------------------------------------------------------------------- checks, launches
def _ptr(t):
    return None if t is None else t.data_ptr()


def _act(t, name, ndim=None, like=None):
    """An activation tensor: on a device, of a known type (of `like`'s type and device where given)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor (got {type(t).__name__})")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor (got {t.device}); the sequence operators have no CPU path")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: dtype {t.dtype}, expected float32, bfloat16 or float16")
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError(f"{name}: dtype {t.dtype}, expected {like.dtype} as the other activations")
        if t.device != like.device:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {like.device}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {ndim} dimensions")
    return t


def _shaped(t, shape, name):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {list(shape)}")
    return t


def _weight(t, shape, name, device):
    """A parameter, used in fp32 and contiguous (a differentiable cast: its gradient comes back in its own type)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_floating_point():
        raise TypeError(f"{name} must be a floating tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    return _shaped(t, shape, name).to(torch.float32).contiguous()


def _marks(t, shape, name, device):
    """starts / reset: bytes or truth values."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.uint8, torch.bool):
        raise TypeError(f"{name} must be a uint8 or bool tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    t = _shaped(t, shape, name).contiguous()
    return t.view(torch.uint8) if t.dtype == torch.bool else t


def _lines(t):
    """t with a contiguous last dimension."""
    return t if t is None or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _no_grad_needed(name, *ts):
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in ts):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")


def _call(name, device, *args):
    """One entry point of libpnp on `device`'s current stream."""
    f = getattr(_lib.load(), name)
    stream = C.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    if device.index == torch.cuda.current_device():
        rc = f(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = f(*args, stream)
    if rc:
        _lib.check(rc, name)


def _floats(name, desc):
    """A workspace size that an entry point reports."""
    n = getattr(_lib.load(), name)(C.byref(desc))
    if n < 0:
        _lib.check(int(n), name)
    return int(n)


def _scratch(n, device):
    return torch.empty(n, dtype=torch.float32, device=device) if n else None


# ---------------------------------------------------------------------------------- norm
def _norm_desc(x, residual, weight, eps):
    d = _lib.PnpNormDesc()
    d.rows, d.dim, d.type, d.eps = x.shape[0], x.shape[1], _TYPES[x.dtype], eps
    d.res_type = _TYPES[(x if residual is None else residual).dtype]
    d.x, d.x_stride, d.weight = x.data_ptr(), x.stride(0), weight.data_ptr()
    if residual is not None:
        d.residual, d.r_stride = residual.data_ptr(), residual.stride(0)
    return d


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, train):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        s = x if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
        rstd = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if train else None
        d = _norm_desc(x, residual, weight, eps)
        d.y, d.rstd = y.data_ptr(), _ptr(rstd)
        if residual is not None:
            d.s = s.data_ptr()
        _call("pnp_rms_norm", x.device, C.byref(d))
        if train:
            ctx.save_for_backward(s, weight, rstd)
            ctx.xtype, ctx.added = x.dtype, residual is not None
            ctx.set_materialize_grads(False)
        return y, (s.view_as(s) if residual is None else s)   # (the stream goes on through here: one rounding of dx + ds)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        s, weight, rstd = ctx.saved_tensors
        if dy is None:
            if ds is None:
                return None, None, None, None, None
            return ds.to(ctx.xtype), ds if ctx.added else None, None, None, None
        dy, ds = _lines(dy), _lines(ds)
        d = _lib.PnpNormBwdDesc()
        d.rows, d.dim, d.type, d.res_type = s.shape[0], s.shape[1], _TYPES[ctx.xtype], _TYPES[s.dtype]
        d.dy, d.dy_stride, d.s, d.s_stride = dy.data_ptr(), dy.stride(0), s.data_ptr(), s.stride(0)
        if ds is not None:
            d.ds, d.ds_stride = ds.data_ptr(), ds.stride(0)
        d.weight, d.rstd = weight.data_ptr(), rstd.data_ptr()
        dx = torch.empty(s.shape, dtype=ctx.xtype, device=s.device)
        d.dx, dres = dx.data_ptr(), dx
        if s.dtype != ctx.xtype:
            dres = torch.empty(s.shape, dtype=s.dtype, device=s.device)
            d.dres = dres.data_ptr()
        dw = None
        if ctx.needs_input_grad[2]:
            dw = torch.empty_like(weight)
            n = _floats("pnp_rms_norm_bwd_workspace", d)
            ws = _scratch(n, s.device)
            d.dweight, d.workspace, d.workspace_floats = dw.data_ptr(), _ptr(ws), n
        _call("pnp_rms_norm_bwd", s.device, C.byref(d))
        return dx, dres if ctx.added else None, dw, None, None


def _norm_inputs(x, weight, residual, eps):
    _act(x, "x")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x: shape {tuple(x.shape)}, expected [..., dim] with dim > 0")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    dim = x.shape[-1]
    if weight is None:
        raise TypeError("weight must be a floating tensor")
    weight = _weight(weight, (dim,), "weight", x.device)
    if residual is not None:
        _act(residual, "residual")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"residual: dtype {residual.dtype}, expected {x.dtype} or float32")
        if residual.device != x.device:
            raise ValueError(f"residual is on {residual.device}, the other tensors on {x.device}")
        residual = _lines(_shaped(residual, x.shape, "residual").reshape(-1, dim))
    return _lines(x.reshape(-1, dim)), weight, residual


def add_rms_norm(x, weight, residual=None, eps=1e-6):
    """``s = x + residual``, ``y = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension;
    returns ``(y, s)``.  ``s`` is held in the residual's type (x's, or fp32 under 16-bit activations:
    a residual stream that many layers add to), and what is held is what is normalised; without a
    residual ``s`` is ``x``.  A row that holds infinity or NaN is NaN in ``y``."""
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x2, weight, r2 = _norm_inputs(x, weight, residual, eps)
    train = torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad or (r2 is not None and r2.requires_grad))
    y, s = _AddRmsNorm.apply(x2, r2, weight, eps, train)
    return y.view(shape), s.view(shape) if train or r2 is not None else x


def _q8_out(x2):
    """8-bit rows, 16 bytes apart at least: the product's loads want rows on 16-byte boundaries."""
    rows, dim = x2.shape
    q = torch.empty(rows, -(-dim // 16) * 16, dtype=torch.int8, device=x2.device)
    return q, torch.empty(rows, dtype=torch.float32, device=x2.device)


def _q8_view(q, scale, shape):
    return q.view(*shape[:-1], q.shape[1])[..., :shape[-1]], scale.view(shape[:-1])


def add_rms_norm_q8(x, weight, residual=None, eps=1e-6):
    """``add_rms_norm`` with its output in 8 bits: returns ``(q, scale, s)``, ``y ~ q * scale[..., None]``
    with ``scale = max|y| / 127`` of the row (0 for a row of zeros; NaN, and q 0, where the row holds
    infinity or NaN) and q rounded to nearest even from the unrounded y.  For serving: no gradient."""
    _no_grad_needed("add_rms_norm_q8", x, weight, residual)
    shape = x.shape if isinstance(x, torch.Tensor) else None
    x2, weight, r2 = _norm_inputs(x, weight, residual, eps)
    q, scale = _q8_out(x2)
    d = _norm_desc(x2, r2, weight, eps)
    d.q, d.q_stride, d.scale = q.data_ptr(), q.stride(0), scale.data_ptr()
    s = x
    if r2 is not None:
        s = torch.empty(shape, dtype=r2.dtype, device=x.device)
        d.s = s.data_ptr()
    _call("pnp_rms_norm", x.device, C.byref(d))
    return (*_q8_view(q, scale, shape), s)


def quantize_rows(x):
    """Rows (the last dimension) in 8 bits: ``(q, scale)`` with ``scale = max|x| / 127`` of each row, as
    ``add_rms_norm_q8`` does.  A weight [N, K] of ``matmul_i8`` is quantised by it once, an activation per
    token.  For serving: no gradient."""
    _no_grad_needed("quantize_rows", x)
    _act(x, "x")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x: shape {tuple(x.shape)}, expected [..., dim] with dim > 0")
    x2 = _lines(x.reshape(-1, x.shape[-1]))
    q, scale = _q8_out(x2)
    _call("pnp_quantize_rows", x.device, x2.data_ptr(), x2.stride(0), _TYPES[x.dtype], x2.shape[0], x2.shape[1], q.data_ptr(),
          q.stride(0), scale.data_ptr())
    return _q8_view(q, scale, x.shape)


# ---------------------------------------------------------------------------------- product in 8 bits
def matmul_i8(q, scale, wq, wscale, bias=None, out_dtype=torch.float32):
    """``out[..., n] = sum_k q[..., k] wq[n, k] * scale[...] * wscale[n] + bias[n]``: q [..., K] and wq
    [N, K] in int8, the sum exact (32-bit integers; K up to 131071), scaled in fp32 and rounded once to
    ``out_dtype``.  For serving: no gradient."""
    _no_grad_needed("matmul_i8", scale, wscale, bias)
    for t, name in ((q, "q"), (wq, "wq")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int8:
            raise TypeError(f"{name} must be an int8 tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a device tensor (got {t.device}); the sequence operators have no CPU path")
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype {out_dtype}, expected float32, bfloat16 or float16")
    if wq.dim() != 2 or q.dim() < 1 or q.shape[-1] != wq.shape[1] or 0 in wq.shape:
        raise ValueError(f"q {tuple(q.shape)} and wq {tuple(wq.shape)}: expected [..., K] and [N, K]")
    if wq.device != q.device:
        raise ValueError(f"wq is on {wq.device}, the other tensors on {q.device}")
    K, N = wq.shape[1], wq.shape[0]
    scale = _weight(scale, q.shape[:-1], "scale", q.device)
    wscale = _weight(wscale, (N,), "wscale", q.device)
    bias = _weight(bias, (N,), "bias", q.device)
    if scale is None or wscale is None:
        raise TypeError("scale and wscale must be floating tensors")
    q2, wq = _i8_rows(q.reshape(-1, K)), _i8_rows(wq)
    out = torch.empty(*q.shape[:-1], N, dtype=out_dtype, device=q.device)
    d = _lib.PnpI8Desc()
    d.M, d.N, d.K, d.out_type = q2.shape[0], N, K, _TYPES[out_dtype]
    d.q, d.q_stride, d.wq, d.wq_stride = q2.data_ptr(), max(q2.stride(0), K), wq.data_ptr(), max(wq.stride(0), K)
    d.scale, d.wscale, d.bias, d.out = scale.data_ptr(), wscale.data_ptr(), _ptr(bias), out.data_ptr()
    _call("pnp_matmul_i8", q.device, C.byref(d))
    return out


def _i8_rows(t):
    """Rows that do not overlap, contiguous each (a broadcast row is copied out)."""
    t = _lines(t)
    return t if t.shape[0] <= 1 or t.stride(0) >= t.shape[1] else t.contiguous()


# ---------------------------------------------------------------------------------- causal convolution
def _conv_desc(x, weight, bias, silu, starts, state):
    d = _lib.PnpConvDesc()
    d.B, d.L, d.dim, d.width = x.shape[0], x.shape[1], x.shape[2], weight.shape[1]
    d.type, d.silu = _TYPES[x.dtype], int(silu)
    d.x, d.x_bstride, d.x_tstride = x.data_ptr(), x.stride(0), x.stride(1)
    d.weight, d.bias, d.starts, d.state = weight.data_ptr(), _ptr(bias), _ptr(starts), _ptr(state)
    return d


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, starts, state, train):
        B, L, D = x.shape
        y = torch.empty(B, L, D, dtype=x.dtype, device=x.device)
        last = torch.empty(B, weight.shape[1] - 1, D, dtype=x.dtype, device=x.device)
        d = _conv_desc(x, weight, bias, silu, starts, state)
        d.y, d.last_state = y.data_ptr(), last.data_ptr()
        _call("pnp_causal_conv", x.device, C.byref(d))
        if train:
            ctx.save_for_backward(x, weight, bias, starts, state)
            ctx.silu = silu
            ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, starts, state = ctx.saved_tensors
        if dy is None and dlast is None:
            return (None,) * 7
        dy = torch.zeros_like(x) if dy is None else _lines(dy)
        d = _lib.PnpConvBwdDesc()
        d.f = _conv_desc(x, weight, bias, ctx.silu, starts, state)
        d.dy, d.dy_bstride, d.dy_tstride = dy.data_ptr(), dy.stride(0), dy.stride(1)
        if dlast is not None:
            dlast = dlast.contiguous()
            d.dlast = dlast.data_ptr()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d.dx = dx.data_ptr()
        dw = db = dstate = None
        if ctx.needs_input_grad[1]:
            dw = torch.empty_like(weight)
            d.dweight = dw.data_ptr()
        if bias is not None and ctx.needs_input_grad[2]:
            db = torch.empty_like(bias)
            d.dbias = db.data_ptr()
        if state is not None and ctx.needs_input_grad[5]:
            dstate = torch.empty_like(state)
            d.dstate = dstate.data_ptr()
        if dw is not None or db is not None:
            n = _floats("pnp_causal_conv_bwd_workspace", d)
            ws = _scratch(n, x.device)
            d.workspace, d.workspace_floats = _ptr(ws), n
        _call("pnp_causal_conv_bwd", x.device, C.byref(d))
        return dx, dw, db, None, None, dstate, None


def _conv_weight(weight, bias, dim, device):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        raise ValueError("weight: expected [dim, width] with a width of 2, 3 or 4")
    return _weight(weight, (dim, weight.shape[1]), "weight", device), _weight(bias, (dim,), "bias", device)


def _silu(activation):
    if activation not in (None, "silu"):
        raise ValueError(f"activation {activation!r}, expected None or 'silu'")
    return activation == "silu"


def causal_conv(x, weight, bias=None, activation=None, starts=None, state=None):
    """``pre[b, t, d] = bias[d] + sum_j weight[d, j] x[b, t - W + 1 + j, d]`` with W 2, 3 or 4, and
    ``pre * sigmoid(pre)`` where ``activation`` is "silu"; x [B, L, D].  What lies before t = 0 comes from
    ``state`` [B, W - 1, D] (x's type; zeros without one).  Returns ``(y, last_state)``: the last W - 1
    tokens of the sequence that goes on (zeros before its start), for the next call or for
    ``causal_conv_step``.  ``starts``: see the module's text."""
    _act(x, "x", 3)
    if x.shape[2] == 0:
        raise ValueError("x: no channels")
    silu = _silu(activation)
    weight, bias = _conv_weight(weight, bias, x.shape[2], x.device)
    starts = _marks(starts, x.shape[:2], "starts", x.device)
    if state is not None:
        state = _shaped(_act(state, "state", 3, like=x), (x.shape[0], weight.shape[1] - 1, x.shape[2]), "state").contiguous()
    x = _lines(x)
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state))
    return _CausalConv.apply(x, weight, bias, silu, starts, state, train)


def causal_conv_step(x, state, weight, bias=None, activation=None, reset=None):
    """One token of each of B sequences: x [B, D] -> y [B, D], ``state`` [B, W - 1, D] (contiguous, x's
    type) advanced in place.  ``reset`` [B] (uint8 or bool) nonzero: that sequence begins at this token.
    For serving: no gradient."""
    _no_grad_needed("causal_conv_step", x, state, weight, bias)
    _act(x, "x", 2)
    if x.shape[1] == 0:
        raise ValueError("x: no channels")
    silu = _silu(activation)
    weight, bias = _conv_weight(weight, bias, x.shape[1], x.device)
    W = weight.shape[1]
    _shaped(_act(state, "state", 3, like=x), (x.shape[0], W - 1, x.shape[1]), "state")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is advanced in place")
    reset = _marks(reset, x.shape[:1], "reset", x.device)
    x = _lines(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _call("pnp_causal_conv_step", x.device, x.data_ptr(), x.stride(0), state.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(reset),
          x.shape[0], x.shape[1], W, _TYPES[x.dtype], int(silu), y.data_ptr())
    return y


# ---------------------------------------------------------------------------------- selective scan
def _scan_desc(u, delta, A, Bm, Cm, D, z, delta_bias, starts, state):
    d = _lib.PnpScanDesc()
    d.B, d.L, d.dim, d.N, d.groups, d.type = u.shape[0], u.shape[1], u.shape[2], A.shape[1], Bm.shape[2], _TYPES[u.dtype]
    for name, short, t in (("u", "u", u), ("delta", "delta", delta), ("z", "z", z), ("Bm", "B", Bm), ("Cm", "C", Cm)):
        if t is not None:
            setattr(d, name, t.data_ptr())
            setattr(d, short + "_bstride", t.stride(0))
            setattr(d, short + "_tstride", t.stride(1))
    d.A, d.D, d.delta_bias, d.state, d.starts = A.data_ptr(), _ptr(D), _ptr(delta_bias), _ptr(state), _ptr(starts)
    return d


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, Bm, Cm, D, z, delta_bias, starts, state, train):
        out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        last = torch.empty(u.shape[0], u.shape[2], A.shape[1], dtype=torch.float32, device=u.device)
        d = _scan_desc(u, delta, A, Bm, Cm, D, z, delta_bias, starts, state)
        d.out, d.last_state = out.data_ptr(), last.data_ptr()
        n = _floats("pnp_scan_workspace", d)
        ws = _scratch(n, u.device)
        d.workspace, d.workspace_floats = _ptr(ws), n
        ckpt = None
        if train:
            n = _floats("pnp_scan_ckpt_floats", d)
            ckpt = torch.empty(n, dtype=torch.float32, device=u.device)
            d.ckpt, d.ckpt_floats = ckpt.data_ptr() if n else None, n
        _call("pnp_selective_scan", u.device, C.byref(d))
        if train:
            ctx.save_for_backward(u, delta, A, Bm, Cm, D, z, delta_bias, starts, state, ckpt)
            ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        u, delta, A, Bm, Cm, D, z, delta_bias, starts, state, ckpt = ctx.saved_tensors
        if dout is None and dlast is None:
            return (None,) * 11
        dev = u.device
        dout = torch.zeros_like(u) if dout is None else _lines(dout)
        d = _lib.PnpScanBwdDesc()
        d.f = _scan_desc(u, delta, A, Bm, Cm, D, z, delta_bias, starts, state)
        d.f.ckpt, d.f.ckpt_floats = ckpt.data_ptr() if ckpt.numel() else None, ckpt.numel()
        d.dout, d.dout_bstride, d.dout_tstride = dout.data_ptr(), dout.stride(0), dout.stride(1)
        if dlast is not None:
            dlast = dlast.contiguous()
            d.dlast = dlast.data_ptr()
        du, ddelta = (torch.empty(u.shape, dtype=u.dtype, device=dev) for _ in range(2))
        dz = None if z is None else torch.empty(u.shape, dtype=u.dtype, device=dev)
        dB, dC = (torch.empty(Bm.shape, dtype=u.dtype, device=dev) for _ in range(2))
        dA = torch.empty_like(A)
        dD = None if D is None else torch.empty_like(D)
        dbias = None if delta_bias is None else torch.empty_like(delta_bias)
        dstate = None if state is None else torch.empty_like(state)
        d.du, d.ddelta, d.dz, d.dB, d.dC = du.data_ptr(), ddelta.data_ptr(), _ptr(dz), dB.data_ptr(), dC.data_ptr()
        d.dA, d.dD, d.ddelta_bias, d.dstate = dA.data_ptr(), _ptr(dD), _ptr(dbias), _ptr(dstate)
        n = _floats("pnp_scan_bwd_workspace", d)
        ws = _scratch(n, dev)
        d.workspace, d.workspace_floats = _ptr(ws), n
        _call("pnp_selective_scan_bwd", dev, C.byref(d))
        return du, ddelta, dA, dB, dC, dD, dz, dbias, None, dstate, None


def _scan_inputs(u, delta, A, B, C_, D, z, delta_bias, lead):
    """Checks of what the scan and its step share; lead: dimensions before the channels."""
    _act(u, "u", lead + 1)
    dim = u.shape[-1]
    if dim == 0:
        raise ValueError("u: no channels")
    _shaped(_act(delta, "delta", like=u), u.shape, "delta")
    if z is not None:
        _shaped(_act(z, "z", like=u), u.shape, "z")
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        raise ValueError("A: expected [dim, N] with N from 1 to 64")
    A = _weight(A, (dim, A.shape[1]), "A", u.device)
    _act(B, "B", like=u)
    _act(C_, "C", like=u)
    if B.dim() == lead + 1 and C_.dim() == lead + 1:
        B, C_ = B.unsqueeze(-2), C_.unsqueeze(-2)
    groups = B.shape[-2] if B.dim() == lead + 2 else 0
    want = (*u.shape[:-1], groups, A.shape[1])
    if groups < 1 or dim % groups or tuple(B.shape) != want or tuple(C_.shape) != want:
        raise ValueError(f"B {tuple(B.shape)} and C {tuple(C_.shape)}: expected [{', '.join(map(str, u.shape[:-1]))}, "
                         f"(groups,) {A.shape[1]}] with groups dividing {dim}")
    D, delta_bias = _weight(D, (dim,), "D", u.device), _weight(delta_bias, (dim,), "delta_bias", u.device)
    return _lines(u), _lines(delta), A, _groups(B), _groups(C_), D, _lines(z), delta_bias


def _groups(t):
    """[..., groups, N] with both of the last dimensions contiguous."""
    if t.shape[-1] > 1 and t.stride(-1) != 1 or t.shape[-2] > 1 and t.stride(-2) != t.shape[-1]:
        return t.contiguous()
    return t


def _state32(state, shape, device):
    if not isinstance(state, torch.Tensor) or state.dtype != torch.float32:
        raise TypeError("state must be a float32 tensor")
    if state.device != device:
        raise ValueError(f"state is on {state.device}, the other tensors on {device}")
    return _shaped(state, shape, "state")


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, starts=None, state=None):
    """``dt = softplus(delta + delta_bias)``, ``h[t] = exp(dt A) h[t - 1] + dt u B``, ``y = sum_n C h + D u``,
    ``out = y * z * sigmoid(z)`` (y without a z).  u, delta, z [B, L, dim]; A [dim, N], N up to 64; B, C
    [B, L, N], or [B, L, groups, N] where each ``dim / groups`` neighbouring channels share a group; D and
    delta_bias [dim].  h before t = 0 is ``state`` [B, dim, N] in fp32 (zeros without one).  Returns
    ``(out, last_state)``, the state in fp32 for the next call or for ``selective_scan_step``.
    ``starts``: see the module's text."""
    u, delta, A, B, C, D, z, delta_bias = _scan_inputs(u, delta, A, B, C, D, z, delta_bias, 2)
    starts = _marks(starts, u.shape[:2], "starts", u.device)
    if state is not None:
        state = _state32(state, (u.shape[0], u.shape[2], A.shape[1]), u.device).contiguous()
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (u, delta, A, B, C, D, z, delta_bias, state))
    return _SelectiveScan.apply(u, delta, A, B, C, D, z, delta_bias, starts, state, train)


def selective_scan_step(u, state, delta, A, B, C, D=None, z=None, delta_bias=None, reset=None):
    """One token of each of B sequences: u, delta, z [B, dim], B, C [B, N] or [B, groups, N] -> out [B, dim],
    ``state`` [B, dim, N] (fp32, contiguous) advanced in place.  ``reset`` [B] (uint8 or bool) nonzero: that
    sequence begins at this token.  For serving: no gradient."""
    _no_grad_needed("selective_scan_step", u, state, delta, A, B, C, D, z, delta_bias)
    u, delta, A, B, C, D, z, delta_bias = _scan_inputs(u, delta, A, B, C, D, z, delta_bias, 1)
    _state32(state, (u.shape[0], u.shape[1], A.shape[1]), u.device)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is advanced in place")
    reset = _marks(reset, u.shape[:1], "reset", u.device)
    out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    d = _lib.PnpScanDesc()
    d.B, d.L, d.dim, d.N, d.groups, d.type = u.shape[0], 1, u.shape[1], A.shape[1], B.shape[1], _TYPES[u.dtype]
    for name, short, t in (("u", "u", u), ("delta", "delta", delta), ("z", "z", z), ("Bm", "B", B), ("Cm", "C", C)):
        if t is not None:
            setattr(d, name, t.data_ptr())
            setattr(d, short + "_bstride", t.stride(0))
    d.A, d.D, d.delta_bias, d.state, d.last_state = A.data_ptr(), _ptr(D), _ptr(delta_bias), state.data_ptr(), state.data_ptr()
    d.starts, d.out = _ptr(reset), out.data_ptr()
    _call("pnp_selective_scan_step", u.device, _byref(d))
    return out
