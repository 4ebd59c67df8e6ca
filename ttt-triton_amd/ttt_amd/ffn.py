"""The gated feed-forward projections on the HIP path (ttt_ffn_* in include/ttt_amd.h):
both products, the activation and the gating in one kernel, with its backward.

fp32, bf16 or fp16, weights and biases in x's type.  Sums are fp32.  The backward forms
both projections again in place of keeping them; in 16 bits it rounds their gradients to
that type where the gradients of x and of the weights read them (those of the biases are
their sums before).  In fp16 those past its largest number are kept apart, scaled, with as
many bits: a gradient is infinite only where it is itself past it.

A value that is not finite reaches what is formed of it and no other row of x or of the weights.
In fp32, whose values are multiplied in bf16 planes, one above 3.39e38 counts as infinite, and
what an infinite one reaches is NaN."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._common import check_device, dtype_code, on_device
from .ssm import _bytes, _empty, _opt, _rows, _stream, _wants_grad, _whole

MAX_WIDTH = 1 << 20
FEW_ROWS = 64  # up to which the forward reads x and the weights at any alignment
_FAR = 4 << 20  # bytes between x's rows up to which they are read in place


def _ffn_args(x, w_gate, w_up, b_gate, b_up, activation):
    """(device, code of x, (rows, D, F), activation code)"""
    shape, act = x.shape, x.dtype
    D = shape[-1] if shape else 0
    if w_gate.dim() != 2 or w_gate.shape[1] != D or w_up.shape != w_gate.shape:
        raise ValueError(f"w_gate and w_up must be [F,D]=[F,{D}], got {list(w_gate.shape)} and {list(w_up.shape)}")
    F = w_gate.shape[0]
    if not 1 <= D <= MAX_WIDTH or not 1 <= F <= MAX_WIDTH:
        raise ValueError(f"widths must be from 1 to {MAX_WIDTH}, got D={D} and F={F}")
    for n, b in (("b_gate", b_gate), ("b_up", b_up)):
        if b is not None and b.shape != (F,):
            raise ValueError(f"{n} must be [F]=[{F}], got {list(b.shape)}")
    if activation not in _lib.GATE_ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} (one of {tuple(_lib.GATE_ACTIVATIONS)})")
    code, dev, near = dtype_code(act), x.device, x.device.type == "cuda"
    for t in (w_gate, w_up, b_gate, b_up):
        if t is not None:
            if t.dtype != act:
                raise ValueError(f"weights and biases must have x's dtype {act}, got {t.dtype}")
            near = near and t.device == dev
    if not near:
        check_device(x, *[t for t in (w_gate, w_up, b_gate, b_up) if t is not None])
    R = x.numel() // D
    if R >= (1 << 31) - 256:
        raise ValueError(f"gated_linear takes fewer than 2^31 - 256 rows, got {R}")
    return dev, code, (R, D, F), _lib.GATE_ACTIVATIONS[activation]


def _operands(x, w_gate, w_up, b_gate, b_up, sizes, any_rows):
    """(x, its row stride, the weights and biases) as the kernels take them"""
    _, D, _ = sizes
    es = x.element_size()
    align = es if any_rows or es == 4 or D % 8 else 16
    xr, ldx = _rows(x, x.dim() - 1, align, D)
    if align == 16 and ldx * es > _FAR:
        xr, ldx = x.detach().contiguous(), D
    return xr, ldx, _whole(w_gate, align), _whole(w_up, align), _whole(b_gate, es), _whole(b_up, es)


def _ffn_forward(x, w_gate, w_up, b_gate, b_up, activation):
    """(y, sizes and codes)"""
    dev, code, sizes, act = _ffn_args(x, w_gate, w_up, b_gate, b_up, activation)
    R, D, F = sizes
    xr, ldx, wg, wu, bg, bu = _operands(x, w_gate, w_up, b_gate, b_up, sizes, R <= FEW_ROWS)
    y = x.new_empty((*x.shape[:-1], F))
    nws = _bytes("ttt_ffn_workspace_bytes", R, D, F, code)
    ws = torch.empty(nws, device=dev, dtype=torch.uint8) if nws else None
    with on_device(dev):
        st = _lib.load().ttt_ffn_fwd(xr.data_ptr(), ldx, wg.data_ptr(), wu.data_ptr(), _opt(bg), _opt(bu), R, D, F, act, code,
                                     y.data_ptr(), _opt(ws), nws, _stream(dev))
    _lib.check(st, "ttt_ffn_fwd")
    return y, (sizes, code, act)


class GatedLinearFunction(torch.autograd.Function):
    """apply(x, w_gate, w_up, b_gate, b_up, activation) -> y; differentiable wrt all tensors."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation):
        y, ctx.how = _ffn_forward(x, w_gate, w_up, b_gate, b_up, activation)
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, *params = ctx.saved_tensors
        sizes, code, act = ctx.how
        R, D, F = sizes
        dev, needs = x.device, ctx.needs_input_grad
        xr, ldx, wg, wu, bg, bu = _operands(x, *params, sizes, False)
        dyr, ldy = _rows(dy if dy.dtype == x.dtype else dy.to(x.dtype), dy.dim() - 1, x.element_size(), F)
        dx = x.new_empty(x.shape) if needs[0] else None
        dwg, dwu = x.new_empty((2, F, D)) if needs[1] or needs[2] else (None, None)
        dbg, dbu = (x.new_empty(F) if t is not None and n else None for t, n in ((bg, needs[3]), (bu, needs[4])))
        nws = _bytes("ttt_ffn_bwd_workspace_bytes", R, D, F, code)
        ws = torch.empty(nws, device=dev, dtype=torch.uint8)
        with on_device(dev):
            st = _lib.load().ttt_ffn_bwd(xr.data_ptr(), ldx, wg.data_ptr(), wu.data_ptr(), _opt(bg), _opt(bu),
                                         dyr.data_ptr(), ldy, R, D, F, act, code, _opt(dx), _opt(dwg), _opt(dwu),
                                         _opt(dbg), _opt(dbu), ws.data_ptr(), nws, _stream(dev))
        _lib.check(st, "ttt_ffn_bwd")
        return dx, dwg, dwu, dbg, dbu, None


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation: str = "silu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) over the last axis of x [.., D], with
    w_gate and w_up [F,D] and biases [F]: the two projections that a gated feed-forward block
    starts with.  activation: "silu", or "gelu" (a times the normal distribution's integral up
    to a).  Returns [.., F] in x's dtype, which weights and biases share.  x may be columns of
    a wider matrix."""
    if x.dim() and x.numel() == 0 and x.shape[-1]:
        _, _, (_, _, F), _ = _ffn_args(x, w_gate, w_up, b_gate, b_up, activation)
        return _empty(x.new_empty((*x.shape[:-1], F)), x, w_gate, w_up, b_gate, b_up)
    if _wants_grad(x, w_gate, w_up, b_gate, b_up):
        return GatedLinearFunction.apply(x, w_gate, w_up, b_gate, b_up, activation)
    return _ffn_forward(x, w_gate, w_up, b_gate, b_up, activation)[0]


__all__ = ["gated_linear", "GatedLinearFunction"]
