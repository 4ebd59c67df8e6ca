"""Layer norm over the last axis on the HIP path (ttt_layer_norm_* in
include/ttt_amd.h), plain or of a gated input, with its backward.

PostNormFunction (layer_io.py) norms the inner loop's [B,H,NC,K,F] output; this
one takes rows as they are."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._common import as_act, check_device, dtype_code, on_device
from .ssm import _as, _bytes, _empty, _opt, _param, _rows, _stream, _wants_grad, _whole

LAYER_NORM_EPS = 1e-6
MAX_WIDTH = 16384


def _norm_args(x, weight, bias, gate, eps):
    """(device, code of x, weight, bias)"""
    shape, act = x.shape, x.dtype
    D = shape[-1] if shape else 0
    if not 1 <= D <= MAX_WIDTH:
        raise ValueError(f"layer_norm takes rows of 1 to {MAX_WIDTH} values, got {list(shape)}")
    if (weight is None) != (bias is None):
        raise ValueError("layer_norm takes weight and bias, or neither")
    if gate is not None and (gate.shape != shape or gate.dtype != act):
        raise ValueError(f"gate must be as x, {list(shape)} in {act}, got {list(gate.shape)} in {gate.dtype}")
    if not 0.0 < eps <= 1.0:
        raise ValueError(f"eps must be in (0, 1], got {eps}")
    dev = check_device(x, *[t for t in (weight, bias, gate) if t is not None])
    return dev, dtype_code(act), _param(weight, (D,), "weight"), _param(bias, (D,), "bias")


def _norm_forward(x, weight, bias, gate, eps, train):
    """(y, what the backward reads)"""
    dev, code, w, b = _norm_args(x, weight, bias, gate, eps)
    shape, es = x.shape, x.element_size()
    D, lead = shape[-1], len(shape) - 1
    xr, ldx = _rows(x, lead, es, D)
    gr, ldg = (None, 0) if gate is None else _rows(gate, lead, es, D)
    y = x.new_empty(shape)
    R = y.numel() // D
    if R >= 1 << 31:
        raise ValueError(f"layer_norm takes fewer than 2^31 rows, got {R}")
    stats = torch.empty((R, 2), device=dev, dtype=torch.float32) if train else None
    with on_device(dev):
        st = _lib.load().ttt_layer_norm_fwd(xr.data_ptr(), ldx, _opt(gr), ldg, _opt(w), _opt(b), R, D, float(eps), code,
                                            y.data_ptr(), _opt(stats), _stream(dev))
    _lib.check(st, "ttt_layer_norm_fwd")
    return y, (xr, ldx, gr, ldg, w, stats)


class LayerNormFunction(torch.autograd.Function):
    """apply(x, weight, bias, gate, eps) -> y; differentiable wrt all four tensors."""

    @staticmethod
    def forward(ctx, x, weight, bias, gate, eps):
        y, (xr, ldx, gr, ldg, w, stats) = _norm_forward(x, weight, bias, gate, eps, True)
        ctx.save_for_backward(xr, gr, w, stats)
        ctx.lds, ctx.strides = (ldx, ldg), (xr.stride(), None if gr is None else gr.stride())
        ctx.dtypes = None if weight is None else (weight.dtype, bias.dtype)
        ctx.shape = x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, gate, w, stats = ctx.saved_tensors
        dev, dt = x.device, x.dtype
        D = ctx.shape[-1]
        R = stats.shape[0]
        ldx, ldg = ctx.lds
        if (x.stride(), None if gate is None else gate.stride()) != ctx.strides:  # (as in ssm.py)
            x, ldx = _rows(x, len(ctx.shape) - 1, x.element_size(), D)
            if gate is not None:
                gate, ldg = _rows(gate, len(ctx.shape) - 1, x.element_size(), D)
        w, stats = _whole(w), _whole(stats)
        dy = as_act(dy, dt)
        dx = x.new_empty(ctx.shape)
        dg = x.new_empty(ctx.shape) if gate is not None else None
        lib = _lib.load()
        dw = db = part = None
        n = 0
        if w is not None and (ctx.needs_input_grad[1] or ctx.needs_input_grad[2]):
            dw, db = torch.empty((2, D), device=dev, dtype=torch.float32)
            n = _bytes("ttt_layer_norm_partial_bytes", R, D)
            part = torch.empty(n // 4, device=dev, dtype=torch.float32)
        with on_device(dev):
            st = lib.ttt_layer_norm_bwd(x.data_ptr(), ldx, _opt(gate), ldg, _opt(w), stats.data_ptr(),
                                        dy.data_ptr(), R, D, dtype_code(dt), dx.data_ptr(), _opt(dg), _opt(dw),
                                        _opt(db), _opt(part), n, _stream(dev))
        _lib.check(st, "ttt_layer_norm_bwd")
        if dw is not None:
            dw, db = _as(dw, ctx.dtypes[0]), _as(db, ctx.dtypes[1])
        return dx, dw, db, dg, None


def layer_norm(x, weight=None, bias=None, gate=None, eps: float = LAYER_NORM_EPS):
    """(v - mean v) / sqrt(var v + eps) * weight + bias over the last axis (up to
    16,384 values) of v = x, or of v = x * silu(gate) where a gate of x's shape and
    dtype is given.  weight and bias [D], both or neither; the variance is the biased
    one.  x and gate may be columns of a wider matrix."""
    if x.dim() and x.numel() == 0 and x.shape[-1]:
        _norm_args(x, weight, bias, gate, eps)
        return _empty(x, weight, bias, gate)
    if _wants_grad(x, weight, bias, gate):
        return LayerNormFunction.apply(x, weight, bias, gate, eps)
    return _norm_forward(x, weight, bias, gate, eps, False)[0]


__all__ = ["layer_norm", "LayerNormFunction", "LAYER_NORM_EPS"]
