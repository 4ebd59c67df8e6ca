"""The selective state-space operators on the HIP path (ttt_causal_conv_* and
ttt_scan_* in include/ttt_amd.h): the short causal convolution and the scan,
over whole sequences with gradients, and one token at a time on a state.

causal_conv     y[t,c] = act(bias[c] + sum_k weight[c,k] s[t+k,c]) over x [B,L,C], s
                being the W-1 inputs before the first token followed by x
selective_scan  h_t = exp(d_t A) h_{t-1} + d_t x_t (x) B_t,  y_t = h_t C_t + D x_t
                with d = softplus(dt + dt_bias): one decay a head, x [B,L,H,P], B and
                C [B,L,G,N] shared by the H/G heads of a group, h [B,H,P,N] fp32

Activations share one dtype (fp32, bf16 or fp16; dt may be fp32 beside a 16-bit
x); parameters and scan states are fp32.  x, dt, Bm and Cm may be columns of a
wider contiguous matrix of rows: they are read in place where x, Bm and Cm start
on 16 bytes in every row, and from a copy elsewhere.  Results do not depend on
which; nothing of a call depends on another sequence of its batch, but its
rounding may: the length is cut up by the number of sequences and heads.

Sums, states and their products are fp32; in bf16 calls the masked products, the state
that an output reads and the weights of the gradients of B and C are rounded to 2^-17
of themselves where they are multiplied (the outputs to 2^-8).

A token that is not finite reaches the outputs and states of its own sequence from
that token on, and no earlier output.  In the backward it may reach every gradient
of its sequence.  (An fp32 value above 3.39e38, which bf16 would round to infinity,
counts as not finite in the scan.)

Gradients are of the first order and in reverse mode; forward-mode derivatives raise
NotImplementedError."""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._common import as_act, check_device, dtype_code, f32c, on_device

HEAD_DIMS = (32, 64)
MAX_STATE = 128
CONV_WIDTHS = (2, 3, 4)


def _row_stride(t: torch.Tensor, lead: int, width: int):
    """The stride of t's first `lead` axes as rows a fixed stride apart with the rest,
    `width` values, contiguous inside a row; None where t is not laid out so."""
    if t.is_contiguous():
        return width
    shape, strides = t.shape, t.stride()
    if lead == 1 and len(shape) == 3 and strides[2] == 1 and strides[1] == shape[2] and strides[0] >= width:
        return strides[0]  # (the heads of single tokens, columns of a wider matrix)
    inner, ld, step = 1, None, 0
    for i in range(t.dim() - 1, -1, -1):
        n, st = shape[i], strides[i]
        if i >= lead:
            if n != 1 and st != inner:
                return None
            inner *= n
        elif n != 1:
            if ld is None:  # the innermost leading axis of more than one row gives the stride
                ld = step = st
            elif st != step:
                return None
            step *= n
    ld = width if ld is None else ld
    return ld if ld >= width else None


def _rows(t: torch.Tensor, lead: int, align: int, width: int):
    """(t, row stride) with t's first `lead` axes as rows (_row_stride), `align` bytes of
    alignment; a contiguous copy where t is not laid out so."""
    if t.is_contiguous():
        if (t.data_ptr() | width * t.element_size()) % align == 0:
            return t, width
        return t.clone(), width  # (fresh memory starts on more than any of them)
    ld = _row_stride(t, lead, width)
    if ld is not None and (t.data_ptr() | ld * t.element_size()) % align == 0:
        return t, ld
    return t.detach().contiguous(), width


def _token_rows(t, align, width):
    return _rows(t, 1, align, width)


def _sequence_rows(t, align, width):
    return _rows(t, 2, align, width)


def _near_rows(t, align, width):
    """_rows of [B,L,..], copied too where the rows of a chunk are out of a 32-bit offset's reach"""
    r, ld = _rows(t, 2, align, width)
    if ld * t.element_size() >= 1 << 26 and t.shape[1] > 1:
        return _rows(t.detach().contiguous(), 2, align, width)
    return r, ld


# Hooks on saved tensors may bring one back in another layout than it was saved in (a
# contiguous one most often, after a stay on the CPU): the backwards compare the layouts of
# what they unpack with those that they kept, and find rows and strides again where one differs.

def _whole(t, align: int = 1):
    """t as one contiguous block on `align` bytes"""
    if t is None or t.is_contiguous() and t.data_ptr() % align == 0:
        return t
    return _fresh(t.detach())


def _fresh(t):
    """A contiguous copy, whatever t's strides"""
    return t.clone(memory_format=torch.contiguous_format)


def _stream(dev: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


@functools.lru_cache(maxsize=4096)
def _bytes(name: str, *sizes: int) -> int:
    """What a size function of the library says for these sizes."""
    return getattr(_lib.load(), name)(*sizes)


def _as(g, dt):
    """A gradient in its input's type."""
    return g if g is None or g.dtype == dt else g.to(dt)


def _opt(t):
    return None if t is None else t.data_ptr()


def _param(t, shape, name):
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else f32c(t)


def _empty(x, *params):
    """The result over no tokens or values, of x's shape; the parameters' gradients are 0."""
    y = x.clone()
    for t in params:
        if t is not None and t.requires_grad:
            y = y + (t.sum() * 0).to(y.dtype)
    return y


def _has_tangent(*ts) -> bool:
    """Whether forward-mode derivatives are on their way through one of these."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                                  for t in ts)


def _wants_grad(*ts) -> bool:
    """Whether the call goes through its autograd function: for gradients, and for tangents,
    which the function refuses (without it they would be dropped, under no_grad too)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts) or _has_tangent(*ts)


def _no_grad_through(what, *ts):
    if _has_tangent(*ts):
        raise NotImplementedError(f"{what} has no forward-mode derivative")
    if _wants_grad(*ts):
        raise ValueError(f"{what} updates its state in place and has no gradient: call it under torch.no_grad()")


def _sizes(*ns):
    if max(ns) >= 1 << 31:
        raise ValueError(f"sizes must be below 2^31, got {ns}")


def _state_in_place(state, shape, dt, dev, what):
    if state.shape != shape or state.dtype != dt or not state.is_contiguous() or state.device != dev:
        raise ValueError(f"{what}: the state must be contiguous, {list(shape)} in {dt} on {dev}, got "
                         f"{list(state.shape)} in {state.dtype} on {state.device}")


# ---------------------------------------------------------------------------
# short causal convolution
# ---------------------------------------------------------------------------

def _conv_args(x, weight, bias, state, activation, lead):
    shape, of_w = x.shape, weight.shape
    if len(shape) != lead + 1:
        raise ValueError(f"x must be [{'B,L,C' if lead == 2 else 'B,C'}], got {list(shape)}")
    C = shape[-1]
    if len(of_w) != 2 or of_w[0] != C or of_w[1] not in CONV_WIDTHS:
        raise ValueError(f"weight must be [C,W]=[{C},W] with W in {CONV_WIDTHS}, got {list(of_w)}")
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} (None or 'silu')")
    dev = check_device(x, weight, *[t for t in (bias, state) if t is not None])
    _sizes(*shape)
    return dev, dtype_code(x.dtype), C, of_w[1], f32c(weight), _param(bias, (C,), "bias")


def _conv_state(state, shape, dt):
    if state is None:
        return None
    if tuple(state.shape) != shape:
        raise ValueError(f"initial_state must be [B,W-1,C]={list(shape)}, got {list(state.shape)}")
    return state.detach().to(dt).contiguous()


def _conv_forward(x, weight, bias, state, activation, want_last):
    """(y, last state or None, what the backward reads)"""
    dev, code, C, W, w, b = _conv_args(x, weight, bias, state, activation, 2)
    B, L = x.shape[:2]
    xr, ldx = _rows(x, 2, x.element_size(), C)
    s0 = _conv_state(state, (B, W - 1, C), x.dtype)
    y = x.new_empty((B, L, C))
    last = x.new_empty((B, W - 1, C)) if want_last else None
    with on_device(dev):
        st = _lib.load().ttt_causal_conv_fwd(xr.data_ptr(), ldx, _opt(s0), w.data_ptr(), _opt(b), B, L, C, W,
                                             _lib.ACTIVATIONS[activation], code, y.data_ptr(), _opt(last), _stream(dev))
    _lib.check(st, "ttt_causal_conv_fwd")
    return y, last, (xr, ldx, s0, w, b)


class CausalConvFunction(torch.autograd.Function):
    """apply(x, weight, bias, initial_state, activation, want_last) -> (y, last
    state or None); differentiable wrt x, weight, bias and initial_state."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, activation, want_last):
        y, last, (xr, ldx, s0, w, b) = _conv_forward(x, weight, bias, state, activation, want_last)
        ctx.save_for_backward(xr, s0, w, b)
        ctx.ldx, ctx.strides = ldx, xr.stride()
        ctx.activation = activation
        ctx.dtypes = weight.dtype, None if bias is None else bias.dtype, None if state is None else state.dtype
        ctx.shape = (*x.shape, weight.shape[1])
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, s0, w, b = ctx.saved_tensors
        B, L, C, W = ctx.shape
        dev = x.device
        dt = x.dtype
        ldx = ctx.ldx
        if x.stride() != ctx.strides:
            x, ldx = _sequence_rows(x, x.element_size(), C)
        s0, w, b = _whole(s0), _whole(w), _whole(b)
        dy, dlast = None if dy is None else as_act(dy, dt), None if dlast is None else as_act(dlast, dt)
        dx = x.new_empty((B, L, C))
        ds = x.new_empty((B, W - 1, C)) if ctx.needs_input_grad[3] else None
        dw = w.new_empty((C, W))
        db = w.new_empty(C) if ctx.dtypes[1] is not None else None
        lib = _lib.load()
        part = w.new_empty(_bytes("ttt_causal_conv_partial_bytes", B, L, C, W) // 4)
        with on_device(dev):
            st = lib.ttt_causal_conv_bwd(x.data_ptr(), ldx, _opt(s0), w.data_ptr(), _opt(b), _opt(dy), _opt(dlast),
                                         B, L, C, W, _lib.ACTIVATIONS[ctx.activation], dtype_code(dt), dx.data_ptr(),
                                         _opt(ds), dw.data_ptr(), _opt(db), part.data_ptr(), part.numel() * 4,
                                         _stream(dev))
        _lib.check(st, "ttt_causal_conv_bwd")
        wt, bt, sd = ctx.dtypes
        return dx, _as(dw, wt), _as(db, bt), _as(ds, sd), None, None


def causal_conv(x, weight, bias=None, initial_state=None, activation=None, return_final_state: bool = False):
    """The causal convolution of every channel over x [B,L,C] with weight [C,W],
    W in 2..4, from zeros or initial_state [B,W-1,C] (the inputs before the first
    token, oldest first).  activation: None or "silu".  Returns y [B,L,C], and with
    return_final_state the last W-1 inputs [B,W-1,C] as well: the state that
    causal_conv_step and a later call go on from."""
    if x.dim() == 3 and x.numel() == 0:
        _, _, C, W, _, _ = _conv_args(x, weight, bias, initial_state, activation, 2)
        shape = (x.shape[0], W - 1, C)
        _conv_state(initial_state, shape, x.dtype)
        first = x.new_zeros(shape) if initial_state is None else _fresh(initial_state.to(x.dtype))
        y = _empty(x, weight, bias)
        return (y, first) if return_final_state else y
    if _wants_grad(x, weight, bias, initial_state):
        y, last = CausalConvFunction.apply(x, weight, bias, initial_state, activation, return_final_state)
    else:
        y, last, _ = _conv_forward(x, weight, bias, initial_state, activation, return_final_state)
    return (y, last) if return_final_state else y


def causal_conv_step(x, state, weight, bias=None, activation=None):
    """One token x [B,C] of every sequence: returns y [B,C] and moves state
    [B,W-1,C] (contiguous, in x's dtype) up by one in place.  No gradient."""
    _no_grad_through("causal_conv_step", x, state, weight, bias)
    dev, code, C, W, w, b = _conv_args(x, weight, bias, state, activation, 1)
    B = x.shape[0]
    _state_in_place(state, (B, W - 1, C), x.dtype, dev, "causal_conv_step")
    y = x.new_empty((B, C))
    if B == 0:
        return y
    xr, ldx = _rows(x, 1, x.element_size(), C)
    with on_device(dev):
        st = _lib.load().ttt_causal_conv_step(xr.data_ptr(), ldx, state.data_ptr(), w.data_ptr(), _opt(b), B, C, W,
                                              _lib.ACTIVATIONS[activation], code, y.data_ptr(), _stream(dev))
    _lib.check(st, "ttt_causal_conv_step")
    torch.autograd.graph.increment_version(state)
    return y


# ---------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------

def _scan_args(x, dt, A, Bm, Cm, D, dt_bias, state, lead):
    """(device, (B, L, H, P, G, N), code of x, code of dt, A, D, dt_bias)"""
    shape, of_b, act = x.shape, Bm.shape, x.dtype
    if len(shape) != lead + 2:
        raise ValueError(f"x must be [{'B,L,H,P' if lead == 2 else 'B,H,P'}], got {list(shape)}")
    *rows, H, P = shape
    if len(of_b) != lead + 2 or list(of_b[:lead]) != rows or of_b != Cm.shape:
        raise ValueError(f"Bm and Cm must be {[*rows, 'G', 'N']}, got {list(of_b)} and {list(Cm.shape)}")
    G, N = of_b[lead:]
    if P not in HEAD_DIMS:
        raise ValueError(f"the head dim P must be one of {HEAD_DIMS}, got {P}")
    if N % 16 or not 16 <= N <= MAX_STATE:
        raise ValueError(f"the state's width N must be a multiple of 16 up to {MAX_STATE}, got {N}")
    if G < 1 or H % G:
        raise ValueError(f"the {G} groups of Bm and Cm must divide the {H} heads")
    if dt.shape != (*rows, H):
        raise ValueError(f"dt must be {[*rows, H]}, got {list(dt.shape)}")
    if Bm.dtype != act or Cm.dtype != act:
        raise ValueError(f"Bm and Cm must have x's dtype {act}, got {Bm.dtype} and {Cm.dtype}")
    of_dt = dt.dtype
    if of_dt != act and of_dt != torch.float32:
        raise ValueError(f"dt must be in {act} or float32, got {of_dt}")
    if A is None:
        raise ValueError("A is needed")
    dev = check_device(x, dt, A, Bm, Cm, *[t for t in (D, dt_bias, state) if t is not None])
    _sizes(*rows, H)
    code = dtype_code(act)
    return (dev, (rows[0], rows[1] if lead == 2 else 1, H, P, G, N), code, code if of_dt == act else dtype_code(of_dt),
            _param(A, (H,), "A"), _param(D, (H,), "D"), _param(dt_bias, (H,), "dt_bias"))


def _scan_state(h0, shape):
    if h0 is None:
        return None
    if tuple(h0.shape) != shape:
        raise ValueError(f"initial_state must be [B,H,P,N]={list(shape)}, got {list(h0.shape)}")
    return _whole(f32c(h0), 16)


def _scan_rows(x, dt, Bm, Cm, rows, align, sizes):
    """The four inputs and their row strides as the kernels take them: x, Bm and Cm by
    rows(t, align, width)"""
    _, _, H, P, G, N = sizes
    return (*rows(x, align, H * P), *_rows(dt, dt.dim() - 1, dt.element_size(), H), *rows(Bm, align, G * N),
            *rows(Cm, align, G * N))


def _scan_forward(x, dt, A, Bm, Cm, D, dt_bias, h0, softplus, want_last, train):
    """(y, last state or None, what the backward reads)"""
    dev, sizes, code, dcode, a, d, bias = _scan_args(x, dt, A, Bm, Cm, D, dt_bias, h0, 2)
    B, L, H, P, G, N = sizes
    h0 = _scan_state(h0, (B, H, P, N))
    rows = _scan_rows(x, dt, Bm, Cm, _near_rows, 16, sizes)
    xr, ldx, dr, ldd, br, ldb, cr, ldc = rows
    y = x.new_empty((B, L, H, P))
    last = torch.empty((B, H, P, N), device=dev, dtype=torch.float32) if want_last else None
    lib = _lib.load()
    nst = _bytes("ttt_scan_states_bytes", B, L, H, P, N, code) if train else 0
    nws = _bytes("ttt_scan_workspace_bytes", B, L, H, P, N, code)
    states = torch.empty(nst, device=dev, dtype=torch.uint8) if train else None
    ws = torch.empty(nws, device=dev, dtype=torch.uint8) if nws else None
    with on_device(dev):
        st = lib.ttt_scan_fwd(xr.data_ptr(), ldx, dr.data_ptr(), ldd, a.data_ptr(), br.data_ptr(), ldb, cr.data_ptr(),
                              ldc, _opt(d), _opt(bias), _opt(h0), B, L, H, P, G, N, code, dcode, int(softplus),
                              y.data_ptr(), _opt(last), _opt(states), nst, _opt(ws), nws, _stream(dev))
    _lib.check(st, "ttt_scan_fwd")
    return y, last, (rows, a, d, bias, states)


class SelectiveScanFunction(torch.autograd.Function):
    """apply(x, dt, A, Bm, Cm, D, dt_bias, initial_state, dt_softplus, want_last) ->
    (y, last state or None); differentiable wrt all tensors.  The forward keeps the
    states entering its chunks of 64 tokens (32 in fp32, and in fp16 for N > 64)."""

    @staticmethod
    def forward(ctx, x, dt, A, Bm, Cm, D, dt_bias, h0, softplus, want_last):
        y, last, (rows, a, d, bias, states) = _scan_forward(x, dt, A, Bm, Cm, D, dt_bias, h0, softplus, want_last, True)
        ctx.save_for_backward(rows[0], rows[2], rows[4], rows[6], a, d, bias, states)
        xr, ldx, dr, ldd, br, ldb, cr, ldc = rows
        ctx.lds, ctx.strides = (ldx, ldd, ldb, ldc), (xr.stride(), dr.stride(), br.stride(), cr.stride())
        ctx.softplus = softplus
        ctx.shape = (*x.shape, *Bm.shape[2:])
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (A, D, dt_bias, h0))
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, dt, Bm, Cm, a, d, bias, states = ctx.saved_tensors
        B, L, H, P, G, N = ctx.shape
        ldx, ldd, ldb, ldc = ctx.lds
        if ((x.stride(), dt.stride(), Bm.stride(), Cm.stride()) != ctx.strides
                or (x.data_ptr() | Bm.data_ptr() | Cm.data_ptr()) % 16):
            x, ldx, dt, ldd, Bm, ldb, Cm, ldc = _scan_rows(x, dt, Bm, Cm, _near_rows, 16, ctx.shape)
        a, d, bias, states = _whole(a), _whole(d), _whole(bias), _whole(states, 16)
        dev, act = x.device, x.dtype
        code = dtype_code(act)
        dy = torch.zeros((B, L, H, P), device=dev, dtype=act) if dy is None else dy
        dyr, ldy = _near_rows(dy if dy.dtype == act else dy.to(act), 16, H * P)
        dlast = None if dlast is None else _whole(f32c(dlast), 16)
        dx = x.new_empty((B, L, H, P))
        ddt = dt.new_empty((B, L, H))
        dB, dC = x.new_empty((B, L, G, N)), x.new_empty((B, L, G, N))
        dA, dD, dbias = a.new_empty((3, H)).unbind()
        dh0 = a.new_empty((B, H, P, N)) if ctx.needs_input_grad[7] else None
        lib = _lib.load()
        nws = _bytes("ttt_scan_bwd_workspace_bytes", B, L, H, P, G, N, code)
        ws = states.new_empty(nws)
        with on_device(dev):
            st = lib.ttt_scan_bwd(x.data_ptr(), ldx, dt.data_ptr(), ldd, a.data_ptr(), Bm.data_ptr(), ldb, Cm.data_ptr(),
                                  ldc, _opt(d), _opt(bias), dyr.data_ptr(), ldy, _opt(dlast), states.data_ptr(),
                                  states.numel(), B, L, H, P, G, N, code, dtype_code(dt.dtype), int(ctx.softplus),
                                  dx.data_ptr(), ddt.data_ptr(), dA.data_ptr(), dB.data_ptr(), dC.data_ptr(),
                                  _opt(None if d is None else dD), _opt(None if bias is None else dbias), _opt(dh0),
                                  ws.data_ptr(), nws, _stream(dev))
        _lib.check(st, "ttt_scan_bwd")
        dts = ctx.dtypes
        return (dx, ddt, _as(dA, dts[0]), dB, dC, None if d is None else _as(dD, dts[1]),
                None if bias is None else _as(dbias, dts[2]), _as(dh0, dts[3]), None, None)


def selective_scan(x, dt, A, Bm, Cm, D=None, dt_bias=None, initial_state=None, dt_softplus: bool = True,
                   return_final_state: bool = False):
    """The scan of x [B,L,H,P] with steps dt [B,L,H] (softplus(dt + dt_bias), or with
    dt_softplus=False dt + dt_bias itself, >= 0), rates A [H] < 0, Bm and Cm [B,L,G,N]
    and the skip D [H], from zeros or initial_state [B,H,P,N] fp32.  P is 32 or 64,
    N a multiple of 16 up to 128.  Returns y [B,L,H,P] in x's dtype, and with
    return_final_state the last state [B,H,P,N] fp32 as well, which
    selective_scan_step and a later call go on from.  A step of 0 (dt = -inf under
    the softplus) leaves the state as it is."""
    if x.dim() == 4 and x.numel() == 0:
        dev, (B, _, H, P, _, N), *_ = _scan_args(x, dt, A, Bm, Cm, D, dt_bias, initial_state, 2)
        _scan_state(initial_state, (B, H, P, N))
        first = torch.zeros(B, H, P, N, device=dev) if initial_state is None else _fresh(initial_state.float())
        y = _empty(x, dt, A, Bm, Cm, D, dt_bias)
        return (y, first) if return_final_state else y
    if _wants_grad(x, dt, A, Bm, Cm, D, dt_bias, initial_state):
        y, last = SelectiveScanFunction.apply(x, dt, A, Bm, Cm, D, dt_bias, initial_state, bool(dt_softplus),
                                              return_final_state)
    else:
        y, last, _ = _scan_forward(x, dt, A, Bm, Cm, D, dt_bias, initial_state, bool(dt_softplus), return_final_state,
                                   False)
    return (y, last) if return_final_state else y


def selective_scan_step(x, dt, A, Bm, Cm, state, D=None, dt_bias=None, dt_softplus: bool = True):
    """One token of every sequence: x [B,H,P], dt [B,H], Bm and Cm [B,G,N].  Updates
    state [B,H,P,N] (fp32, contiguous) in place and returns y [B,H,P].  No gradient."""
    _no_grad_through("selective_scan_step", x, dt, A, Bm, Cm, state, D, dt_bias)
    dev, sizes, code, dcode, a, d, bias = _scan_args(x, dt, A, Bm, Cm, D, dt_bias, state, 1)
    B, _, H, P, G, N = sizes
    _state_in_place(state, (B, H, P, N), torch.float32, dev, "selective_scan_step")
    y = x.new_empty((B, H, P))
    if B == 0:
        return y
    xr, ldx, dr, ldd, br, ldb, cr, ldc = _scan_rows(x, dt, Bm, Cm, _token_rows, 4 * x.element_size(), sizes)
    with on_device(dev):
        st = _lib.load().ttt_scan_step(xr.data_ptr(), ldx, dr.data_ptr(), ldd, a.data_ptr(), br.data_ptr(), ldb,
                                       cr.data_ptr(), ldc, _opt(d), _opt(bias), state.data_ptr(), B, H, P, G, N, code,
                                       dcode, int(dt_softplus), y.data_ptr(), _stream(dev))
    _lib.check(st, "ttt_scan_step")
    torch.autograd.graph.increment_version(state)
    return y


__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "CausalConvFunction",
           "SelectiveScanFunction"]
