"""Operators of a policy with memory on device tensors: the layers of ``pnp_amd.history`` (and of
any other sequence model a user builds beside it), each by hand-written HIP kernels of libpnp.so
(include/pnp.h, csrc/seq_*.hip); checks, outputs and gradients are wired in native code
(csrc/seq_torch.cpp, _seqops.so), which is what keeps a call's host time small.

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
packed sequences go one after the other in a row.  Padding is a sequence of its own, with outputs of its
own: where weights are trained it holds finite values, since a gradient of zero times NaN is NaN.

Derivatives are reverse-mode gradients, once: a second gradient is an error, and so is an input with a
forward-mode tangent (``NotImplementedError``).

A captured graph may hold any call, its backward pass too; as everywhere in torch, no eager graph of the
same leaves may live while a backward pass is captured (capture over detached copies of the leaves, or
after the eager graphs are gone).
"""
from __future__ import annotations

import ctypes as C
import os

import torch

from . import _lib

EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_seqops.so")
_ENTRIES = ("pnp_last_error", "pnp_rms_norm", "pnp_rms_norm_bwd", "pnp_rms_norm_bwd_workspace", "pnp_quantize_rows", "pnp_matmul_i8",
            "pnp_causal_conv", "pnp_causal_conv_bwd", "pnp_causal_conv_bwd_workspace", "pnp_causal_conv_step", "pnp_selective_scan",
            "pnp_selective_scan_bwd", "pnp_selective_scan_step", "pnp_scan_ckpt_floats", "pnp_scan_workspace", "pnp_scan_bwd_workspace")


def _load():
    """The native front end, bound to the libpnp that the package has loaded."""
    if not os.path.exists(EXT_PATH):
        raise _lib.PnpError(f"_seqops.so not found at {EXT_PATH}; build the HIP extension first "
                            f"(make -C {_lib.CSRC} or __graft_entry__.build())")
    import importlib.util
    spec = importlib.util.spec_from_file_location("_seqops", EXT_PATH)
    ext = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ext)
    L = _lib.load()
    ext.bind({name: C.cast(getattr(L, name), C.c_void_p).value for name in _ENTRIES})
    return ext


class _Lazy:
    """Loads the front end at the first call (importing the package touches no library)."""

    def __getattr__(self, name):
        global _ext
        _ext = _load()
        return getattr(_ext, name)


_ext = _Lazy()


def add_rms_norm(x, weight, residual=None, eps=1e-6):
    """``s = x + residual``, ``y = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension;
    returns ``(y, s)``.  ``s`` is held in the residual's type (x's, or fp32 under 16-bit activations:
    a residual stream that many layers add to), and what is held is what is normalised; without a
    residual ``s`` is ``x`` (take the stream's gradient through it: the two paths then meet in one
    rounding).  A row that holds NaN is NaN in ``y``; in one whose squares outgrow fp32 (infinity among
    them) what is finite is 0 and infinity NaN, as by the formula."""
    return _ext.add_rms_norm(x, weight, residual, eps)


def add_rms_norm_q8(x, weight, residual=None, eps=1e-6):
    """``add_rms_norm`` with its output in 8 bits: returns ``(q, scale, s)``, ``y ~ q * scale[..., None]``
    with ``scale = max|y| / 127`` of the row (0, and q 0, where that is below the least normal fp32, as in a
    row of zeros; NaN, and q 0, where the row holds infinity or NaN) and q the fp32 quotient ``y / scale`` of
    the unrounded y, rounded to nearest even.  For serving: no gradient."""
    return _ext.add_rms_norm_q8(x, weight, residual, eps)


def quantize_rows(x):
    """Rows (the last dimension) in 8 bits: ``(q, scale)`` with ``scale = max|x| / 127`` of each row, as
    ``add_rms_norm_q8`` does.  A weight [N, K] of ``matmul_i8`` is quantised by it once, an activation per
    token.  For serving: no gradient."""
    return _ext.quantize_rows(x)


def matmul_i8(q, scale, wq, wscale, bias=None, out_dtype=torch.float32):
    """``out[..., n] = sum_k q[..., k] wq[n, k] * scale[...] * wscale[n] + bias[n]``: q [..., K] and wq
    [N, K] in int8, the sum exact (32-bit integers; K up to 131071), scaled in fp32 and rounded once to
    ``out_dtype``.  Up to 2^31 rows of q, N up to 2^24, and fewer than 2^23 tiles of 256 x 256 outputs; past
    these a ``PnpError``.  For serving: no gradient."""
    return _ext.matmul_i8(q, scale, wq, wscale, bias, out_dtype)


def causal_conv(x, weight, bias=None, activation=None, starts=None, state=None):
    """``pre[b, t, d] = bias[d] + sum_j weight[d, j] x[b, t - W + 1 + j, d]`` with W 2, 3 or 4, and
    ``pre * sigmoid(pre)`` where ``activation`` is "silu"; x [B, L, D].  What lies before t = 0 comes from
    ``state`` [B, W - 1, D] (x's type; zeros without one).  Returns ``(y, last_state)``: the last W - 1
    tokens of the sequence that goes on (zeros before its start), for the next call or for
    ``causal_conv_step``.  ``starts``: see the module's text.  One launch: calls with B * ceil(L / 8) * D below
    2^32 always fit; one that does not is a ``PnpError``."""
    return _ext.causal_conv(x, weight, bias, activation, starts, state)


def causal_conv_step(x, state, weight, bias=None, activation=None, reset=None):
    """One token of each of B sequences: x [B, D] -> y [B, D], ``state`` [B, W - 1, D] (contiguous, x's
    type) advanced in place (inputs that lie in it are copied first).  ``reset`` [B] (uint8 or bool) nonzero: that
    sequence begins at this token.  For serving: no gradient."""
    return _ext.causal_conv_step(x, state, weight, bias, activation, reset)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, starts=None, state=None):
    """``dt = softplus(delta + delta_bias)``, ``h[t] = exp(dt A) h[t - 1] + dt u B``, ``y = sum_n C h + D u``,
    ``out = y * z * sigmoid(z)`` (y without a z).  u, delta, z [B, L, dim]; A [dim, N], N up to 64; B, C
    [B, L, N], or [B, L, groups, N] where each ``dim / groups`` neighbouring channels share a group; D and
    delta_bias [dim].  h before t = 0 is ``state`` [B, dim, N] in fp32 (zeros without one).  Returns
    ``(out, last_state)``, the state in fp32 for the next call or for ``selective_scan_step``.
    ``starts``: see the module's text.  One launch: B * groups * ceil(dim / groups / C) below 2^24, with C 256,
    128, 64, 32, 16 for N up to 4, 8, 16, 32, 64, and dim * (N + 2) below 2^28 with a gradient; past these a
    ``PnpError``."""
    return _ext.selective_scan(u, delta, A, B, C, D, z, delta_bias, starts, state)


def selective_scan_step(u, state, delta, A, B, C, D=None, z=None, delta_bias=None, reset=None):
    """One token of each of B sequences: u, delta, z [B, dim], B, C [B, N] or [B, groups, N] -> out [B, dim],
    ``state`` [B, dim, N] (fp32, contiguous) advanced in place (inputs that lie in it are copied first).
    ``reset`` [B] (uint8 or bool) nonzero: that sequence begins at this token.  For serving: no gradient."""
    return _ext.selective_scan_step(u, state, delta, A, B, C, D, z, delta_bias, reset)
