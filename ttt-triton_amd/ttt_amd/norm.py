"""Norms over the last axis on the HIP path, with their backwards: layer norm, plain or
of a gated input (ttt_layer_norm_* in include/ttt_amd.h), and the root-mean-square norms
around a block with its gate and residual scale (ttt_block_norm_*).

PostNormFunction (layer_io.py) norms the inner loop's [B,H,NC,K,F] output; this
one takes rows as they are."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._common import as_act, check_device, dtype_code, on_device
from .ssm import _as, _bytes, _empty, _opt, _param, _row_stride, _rows, _stream, _wants_grad, _whole

LAYER_NORM_EPS = 1e-6
MAX_WIDTH = 16384
MAX_BLOCK_WIDTH = 8192  # block_norm's rows


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


# ---------------------------------------------------------------------------
# the norms around a block
# ---------------------------------------------------------------------------

def _block_args(x, weight, residual, gate, scale, next_weight, eps):
    """(device, code of x, code of the residual or -1, the three parameters)"""
    shape, act = x.shape, x.dtype
    D = shape[-1] if shape else 0
    if not 1 <= D <= MAX_BLOCK_WIDTH:
        raise ValueError(f"block_norm takes rows of 1 to {MAX_BLOCK_WIDTH} values, got {list(shape)}")
    code = dtype_code(act)
    if gate is not None and (gate.shape != shape or gate.dtype != act):
        raise ValueError(f"gate must be as x, {list(shape)} in {act}, got {list(gate.shape)} in {gate.dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype not in (act, torch.float32)):
        raise ValueError(f"residual must be {list(shape)} in {act} or float32, got {list(residual.shape)} in "
                         f"{residual.dtype}")
    if next_weight is not None and residual is None:
        raise ValueError("next_weight (the norm before the next block) needs a residual")
    if not 0.0 < eps <= 1.0:
        raise ValueError(f"eps must be in (0, 1], got {eps}")
    dev = x.device
    if dev.type != "cuda":
        check_device(x)
    for t in (weight, residual, gate, scale, next_weight):
        if t is not None and t.device != dev:
            check_device(x, t)
    of = (D,)
    return (dev, code, -1 if residual is None else code if residual.dtype == act else dtype_code(residual.dtype),
            (_param(weight, of, "weight"), _param(scale, of, "scale"), _param(next_weight, of, "next_weight")))


def _block_rows(ts):
    """(the tensors as rows, heads, their row strides): as plain rows where all are laid out
    so, else as wider rows of `heads` each, else from copies."""
    x, *more = ts
    D, dim = x.shape[-1], x.dim()
    if x.is_contiguous() and all(t is None or t.is_contiguous() for t in more):
        return ts, 1, [D if t is not None else 0 for t in ts]
    some = [t for t in ts if t is not None]
    lds = [_row_stride(t, dim - 1, D) for t in some]
    heads = 1
    if None in lds and dim > 2:
        n = some[0].shape[-2]
        wide = [_row_stride(t, dim - 2, n * D) for t in some]
        if sum(ld is None for ld in wide) <= sum(ld is None for ld in lds):
            lds, heads = wide, n
    it = iter(lds)
    rows, strides = [], []
    for t in ts:
        ld = None if t is None else next(it)
        copied = t is not None and ld is None
        rows.append(t.detach().contiguous() if copied else t)
        strides.append(heads * D if copied else ld or 0)
    return rows, heads, strides


def _block_forward(x, weight, residual, gate, scale, next_weight, eps, train):
    """(r, y or None, what the backward reads)"""
    dev, code, rcode, (w, s, w2) = _block_args(x, weight, residual, gate, scale, next_weight, eps)
    shape, D = x.shape, x.shape[-1]
    (xr, gr, rr), heads, (ldx, ldg, ldr) = _block_rows((x, gate, residual))
    r = x.new_empty(shape) if residual is None else residual.new_empty(shape)
    y = None if next_weight is None else x.new_empty(shape)
    R = r.numel() // D
    if R >= 1 << 31:
        raise ValueError(f"block_norm takes fewer than 2^31 rows, got {R}")
    stats = torch.empty((R, 2), device=dev, dtype=torch.float32) if train else None
    with on_device(dev):
        st = _lib.load().ttt_block_norm_fwd(xr.data_ptr(), ldx, _opt(gr), ldg, _opt(rr), ldr, _opt(w), _opt(s), _opt(w2), R,
                                            D, heads, float(eps), code, rcode, r.data_ptr(), _opt(y), _opt(stats),
                                            _stream(dev))
    _lib.check(st, "ttt_block_norm_fwd")
    return r, y, ((xr, gr, rr), heads, (ldx, ldg, ldr), (w, s, w2), stats, (code, rcode))


class BlockNormFunction(torch.autograd.Function):
    """apply(x, weight, residual, gate, scale, next_weight, eps) -> (r, y or None);
    differentiable wrt all six tensors."""

    @staticmethod
    def forward(ctx, x, weight, residual, gate, scale, next_weight, eps):
        r, y, (rows, heads, lds, params, stats, codes) = _block_forward(x, weight, residual, gate, scale, next_weight, eps,
                                                                        True)
        if next_weight is None:  # the sum's gradient alone passes: the residual is not read again
            rows = (*rows[:2], None)
        ctx.save_for_backward(*rows, *params, stats)
        ctx.heads, ctx.lds, ctx.strides = heads, lds, tuple(None if t is None else t.stride() for t in rows)
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (weight, scale, next_weight))
        ctx.shape, ctx.codes = x.shape, codes
        ctx.set_materialize_grads(False)
        return r, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dy):
        x, gate, res, w, s, w2, stats = ctx.saved_tensors
        shape, (code, rcode) = ctx.shape, ctx.codes
        D, R, dev, dt = shape[-1], stats.shape[0], x.device, x.dtype
        heads, (ldx, ldg, ldr) = ctx.heads, ctx.lds
        if tuple(None if t is None else t.stride() for t in (x, gate, res)) != ctx.strides:  # (as in ssm.py)
            (x, gate, res), heads, (ldx, ldg, ldr) = _block_rows((x, gate, res))
        w, s, w2, stats = (_whole(t) for t in (w, s, w2, stats))
        rdt = torch.float32 if rcode == _lib.DTYPE_F32 else dt
        dr, dy = None if dr is None else as_act(dr, rdt), None if dy is None else as_act(dy, dt)
        needs = ctx.needs_input_grad
        # without the next norm r's gradient passes to the residual as it is, and to an x that is
        # neither normed, gated nor scaled
        same = dr if w2 is None and rcode >= 0 else None
        if same is not None and rdt == dt and w is None and s is None and gate is None:
            return same, None, same, None, None, None, None
        dx = x.new_empty(shape)
        dg = x.new_empty(shape) if gate is not None else None
        dres = x.new_empty(shape, dtype=rdt) if rcode >= 0 and needs[2] and same is None else None
        want = [t is not None and needs[i] for t, i in ((w, 1), (s, 4), (w2, 5))]
        dp, part, n = [None] * 3, None, 0
        if any(want):
            dp = [t if q else None for t, q in zip(torch.empty((3, D), device=dev, dtype=torch.float32), want)]
            n = _bytes("ttt_block_norm_partial_bytes", R, D)
            part = torch.empty(n // 4, device=dev, dtype=torch.float32)
        with on_device(dev):
            st = _lib.load().ttt_block_norm_bwd(x.data_ptr(), ldx, _opt(gate), ldg, _opt(res), ldr, _opt(w), _opt(s),
                                                _opt(w2), stats.data_ptr(), _opt(dr), _opt(dy), R, D, heads, code, rcode,
                                                dx.data_ptr(), _opt(dg), _opt(dres), *(_opt(t) for t in dp), _opt(part), n,
                                                _stream(dev))
        _lib.check(st, "ttt_block_norm_bwd")
        dw, ds, dw2 = (None if t is None else _as(t, q) for t, q in zip(dp, ctx.dtypes))
        return dx, dw, dres if same is None else same, dg, ds, dw2, None


def block_norm(x, weight=None, residual=None, gate=None, scale=None, next_weight=None, eps: float = LAYER_NORM_EPS):
    """The norms around a block over the last axis (up to 8,192 values), by root mean squares:

        r = residual + scale * silu(gate) * x / sqrt(mean x^2 + eps) * weight

    each part where it is given (without a weight x is not normed), and, with next_weight and
    a residual, (r, y) with y = r / sqrt(mean r^2 + eps) * next_weight, what the next block
    reads.  gate has x's shape and dtype, the residual x's shape in x's dtype or fp32, which r
    has as well (x's without one); weight, scale and next_weight are [D].  y is normed from r
    before it is rounded; squares are summed in fp32 (rows of a length below 1e19).  x, gate
    and residual may be columns of a wider matrix, by heads too ([.., H, D])."""
    if x.dim() and x.numel() == 0 and x.shape[-1]:
        _block_args(x, weight, residual, gate, scale, next_weight, eps)
        r = _empty(x if residual is None else residual, x, weight, residual, gate, scale, next_weight)
        return r if next_weight is None else (r, _empty(x, weight, residual, gate, scale, next_weight))
    if _wants_grad(x, weight, residual, gate, scale, next_weight):
        r, y = BlockNormFunction.apply(x, weight, residual, gate, scale, next_weight, eps)
    else:
        r, y, _ = _block_forward(x, weight, residual, gate, scale, next_weight, eps, False)
    return r if next_weight is None else (r, y)


__all__ = ["layer_norm", "LayerNormFunction", "block_norm", "BlockNormFunction", "LAYER_NORM_EPS"]
