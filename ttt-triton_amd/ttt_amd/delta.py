"""The gated delta rule on the HIP path (ttt_delta_* in include/ttt_amd.h): over whole
sequences with gradients, and one token at a time on a state.

gated_delta  S_t = e^{g_t} S_{t-1} + u_t (x) k_t,  u_t = beta_t (v_t - e^{g_t} S_{t-1} k_t),
             o_t = scale S_t q_t: what the decayed state misses of v_t at the key k_t is
             written there with weight beta_t.  v [B,L,H,P], q and k [B,L,G,N] shared by the
             H/G heads of a group, g and beta [B,L,H], S [B,H,P,N] fp32

Activations share one dtype (fp32, bf16 or fp16; g and beta may each be fp32 beside a
16-bit v); states are fp32.  q, k, v, g and beta may be columns of a wider contiguous
matrix of rows: they are read in place where q, k and v start on 16 bytes in every row,
and from a copy elsewhere.  Results do not depend on which; nothing of a call depends on
another sequence of its batch, but its rounding may: the length is cut up by the number of
sequences and heads.

Sums, states and their products are fp32; in bf16 calls what leads to bf16 results alone
(the masked products of q and k, the state that an output reads) is rounded to 2^-17 of
itself where it is multiplied (the outputs to 2^-8).

A token whose k, v, g or beta is not finite makes its sequence's outputs (of v: of that
feature's) and states NaN from that token on, and no earlier output; one whose q is not,
its own output.  In the backward it may reach every gradient of its sequence.  (An fp32
value above 3.39e38, which bf16 would round to infinity, counts as not finite.)

Gradients are of the first order and in reverse mode; forward-mode derivatives raise
NotImplementedError."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._common import check_device, dtype_code, f32c, on_device
from .ssm import (_as, _bytes, _empty, _fresh, _near_rows, _no_grad_through, _opt, _rows, _sizes, _state_in_place, _stream,
                  _wants_grad, _whole)

MAX_HEAD_DIM = 256  # P, a multiple of 32
MAX_STATE = 128     # N, a multiple of 16


def _delta_args(q, k, v, g, beta, state, scale, lead):
    """(device, (B, L, H, P, G, N), codes of v, g and beta, scale)"""
    shape, of_k, act = v.shape, k.shape, v.dtype
    if len(shape) != lead + 2:
        raise ValueError(f"v must be [{'B,L,H,P' if lead == 2 else 'B,H,P'}], got {list(shape)}")
    *rows, H, P = shape
    if len(of_k) != lead + 2 or list(of_k[:lead]) != rows or of_k != q.shape:
        raise ValueError(f"q and k must be {[*rows, 'G', 'N']}, got {list(q.shape)} and {list(of_k)}")
    G, N = of_k[lead:]
    if P % 32 or not 32 <= P <= MAX_HEAD_DIM:
        raise ValueError(f"the head dim P must be a multiple of 32 up to {MAX_HEAD_DIM}, got {P}")
    if N % 16 or not 16 <= N <= MAX_STATE:
        raise ValueError(f"the keys' width N must be a multiple of 16 up to {MAX_STATE}, got {N}")
    if G < 1 or H % G:
        raise ValueError(f"the {G} groups of q and k must divide the {H} heads")
    if q.dtype != act or k.dtype != act:
        raise ValueError(f"q and k must have v's dtype {act}, got {q.dtype} and {k.dtype}")
    code = dtype_code(act)
    codes = [code]
    for name, t in (("g", g), ("beta", beta)):
        if t.shape != (*rows, H):
            raise ValueError(f"{name} must be {[*rows, H]}, got {list(t.shape)}")
        if t.dtype != act and t.dtype != torch.float32:
            raise ValueError(f"{name} must be in {act} or float32, got {t.dtype}")
        codes.append(code if t.dtype == act else dtype_code(t.dtype))
    dev = check_device(v, q, k, g, beta, *(() if state is None else (state,)))
    _sizes(*rows, H)
    return (dev, (rows[0], rows[1] if lead == 2 else 1, H, P, G, N), codes, N ** -0.5 if scale is None else float(scale))


def _delta_state(h0, shape):
    if h0 is None:
        return None
    if tuple(h0.shape) != shape:
        raise ValueError(f"initial_state must be [B,H,P,N]={list(shape)}, got {list(h0.shape)}")
    return _whole(f32c(h0), 16)


def _qk_rows(q, k, g, beta, sizes):
    """The four inputs and their row strides as the kernels take them"""
    _, _, H, _, G, N = sizes
    return (*_near_rows(q, 16, G * N), *_near_rows(k, 16, G * N), *_rows(g, 2, g.element_size(), H),
            *_rows(beta, 2, beta.element_size(), H))


def _delta_forward(q, k, v, g, beta, h0, scale, unit, want_last, train):
    """(o, last state or None, what the backward reads)"""
    dev, sizes, codes, scale = _delta_args(q, k, v, g, beta, h0, scale, 2)
    B, L, H, P, G, N = sizes
    code = codes[0]
    h0 = _delta_state(h0, (B, H, P, N))
    rows = _qk_rows(q, k, g, beta, sizes)
    qr, ldq, kr, ldk, gr, ldg, br, ldb = rows
    vr, ldv = _near_rows(v, 16, H * P)
    o = v.new_empty((B, L, H, P))
    last = torch.empty((B, H, P, N), device=dev, dtype=torch.float32) if want_last else None
    lib = _lib.load()
    nsv = _bytes("ttt_delta_saved_bytes", B, L, H, P, N, code) if train else 0
    nws = _bytes("ttt_delta_workspace_bytes", B, L, H, P, N, code)
    if not nws or train and not nsv:  # (0 for what a launch has no threads for)
        raise ValueError(f"gated_delta{' with gradients' if nws else ''} has too many tokens and heads: {list(v.shape)}")
    saved = torch.empty(nsv, device=dev, dtype=torch.uint8) if train else None
    ws = torch.empty(nws, device=dev, dtype=torch.uint8)
    with on_device(dev):
        st = lib.ttt_delta_fwd(qr.data_ptr(), ldq, kr.data_ptr(), ldk, vr.data_ptr(), ldv, gr.data_ptr(), ldg,
                               br.data_ptr(), ldb, _opt(h0), B, L, H, P, G, N, scale, unit, *codes, o.data_ptr(),
                               _opt(last), _opt(saved), nsv, ws.data_ptr(), nws, _stream(dev))
    _lib.check(st, "ttt_delta_fwd")
    return o, last, (rows, saved, ws, sizes, codes, scale)


class GatedDeltaFunction(torch.autograd.Function):
    """apply(q, k, v, g, beta, initial_state, scale, l2_norm, want_last) -> (o, last state
    or None); differentiable wrt all tensors.  The forward keeps the states entering its
    chunks of 64 tokens (32 in fp32 and fp16), what each token's state missed, and its
    workspace: what the chunks' keys and queries give by themselves."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, scale, unit, want_last):
        o, last, (rows, saved, kept, sizes, codes, scale) = _delta_forward(q, k, v, g, beta, h0, scale, unit, want_last, True)
        ctx.save_for_backward(rows[0], rows[2], rows[4], rows[6], saved, kept)
        ctx.lds, ctx.strides = rows[1::2], tuple(t.stride() for t in rows[::2])
        ctx.sizes, ctx.codes, ctx.scale, ctx.unit = sizes, codes, scale, unit
        ctx.state_dtype = None if h0 is None else h0.dtype
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dlast):
        q, k, g, beta, saved, kept = ctx.saved_tensors
        B, L, H, P, G, N = ctx.sizes
        ldq, ldk, ldg, ldb = ctx.lds
        if (q.stride(), k.stride(), g.stride(), beta.stride()) != ctx.strides or (q.data_ptr() | k.data_ptr()) % 16:
            q, ldq, k, ldk, g, ldg, beta, ldb = _qk_rows(q, k, g, beta, ctx.sizes)
        saved, kept = _whole(saved, 16), _whole(kept, 16)
        dev, act = q.device, q.dtype
        do = torch.zeros((B, L, H, P), device=dev, dtype=act) if do is None else do
        dor, ldo = _near_rows(do if do.dtype == act else do.to(act), 16, H * P)
        dlast = None if dlast is None else _whole(f32c(dlast), 16)
        dq, dk = q.new_empty((B, L, G, N)), q.new_empty((B, L, G, N))
        dv = q.new_empty((B, L, H, P))
        dg, db = g.new_empty((B, L, H)), beta.new_empty((B, L, H))
        dh0 = torch.empty((B, H, P, N), device=dev, dtype=torch.float32) if ctx.needs_input_grad[5] else None
        lib = _lib.load()
        nws = _bytes("ttt_delta_bwd_workspace_bytes", B, L, H, P, G, N, ctx.codes[0])
        ws = saved.new_empty(nws)
        with on_device(dev):
            st = lib.ttt_delta_bwd(q.data_ptr(), ldq, k.data_ptr(), ldk, g.data_ptr(), ldg, beta.data_ptr(), ldb,
                                   dor.data_ptr(), ldo, _opt(dlast), saved.data_ptr(), saved.numel(), kept.data_ptr(),
                                   kept.numel(), B, L, H, P, G, N, ctx.scale, ctx.unit, *ctx.codes, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                   dg.data_ptr(), db.data_ptr(), _opt(dh0), ws.data_ptr(), nws, _stream(dev))
        _lib.check(st, "ttt_delta_bwd")
        return dq, dk, dv, dg, db, _as(dh0, ctx.state_dtype), None, None, None


def gated_delta(q, k, v, g, beta, initial_state=None, scale=None, l2_norm: bool = True,
                return_final_state: bool = False):
    """The gated delta rule over v [B,L,H,P] with keys and queries k and q [B,L,G,N],
    log-decays g [B,L,H] (<= 0; -inf forgets the state) and weights beta [B,L,H], from
    zeros or initial_state [B,H,P,N] fp32.  l2_norm: q and k are taken at unit length,
    x / sqrt(|x|^2 + 1e-6), |x|^2 in fp32, for |x| below 1e19 (without it they are used as they are: the state grows without
    bound where beta |k|^2 > 2).  scale: N^-1/2 where none is given.  P is a multiple of 32
    up to 256, N of 16 up to 128.  Returns o [B,L,H,P] in v's dtype, and with
    return_final_state the last state [B,H,P,N] fp32 as well, which gated_delta_step and a
    later call go on from."""
    unit = int(bool(l2_norm))
    if v.dim() == 4 and v.numel() == 0:
        dev, (B, _, H, P, _, N), *_ = _delta_args(q, k, v, g, beta, initial_state, scale, 2)
        _delta_state(initial_state, (B, H, P, N))
        first = torch.zeros(B, H, P, N, device=dev) if initial_state is None else _fresh(initial_state.float())
        o = _empty(v, q, k, g, beta)
        return (o, first) if return_final_state else o
    if _wants_grad(q, k, v, g, beta, initial_state):
        o, last = GatedDeltaFunction.apply(q, k, v, g, beta, initial_state, scale, unit, return_final_state)
    else:
        o, last, _ = _delta_forward(q, k, v, g, beta, initial_state, scale, unit, return_final_state, False)
    return (o, last) if return_final_state else o


def gated_delta_step(q, k, v, g, beta, state, scale=None, l2_norm: bool = True):
    """One token of every sequence: q and k [B,G,N], v [B,H,P], g and beta [B,H].  Updates
    state [B,H,P,N] (fp32, contiguous) in place and returns o [B,H,P].  No gradient."""
    _no_grad_through("gated_delta_step", q, k, v, g, beta, state)
    dev, sizes, codes, scale = _delta_args(q, k, v, g, beta, state, scale, 1)
    B, _, H, P, G, N = sizes
    _state_in_place(state, (B, H, P, N), torch.float32, dev, "gated_delta_step")
    o = v.new_empty((B, H, P))
    if o.numel() == 0:
        return o
    es = v.element_size()
    (qr, ldq), (kr, ldk), (vr, ldv) = _rows(q, 1, 4 * es, G * N), _rows(k, 1, 4 * es, G * N), _rows(v, 1, es, H * P)
    (gr, ldg), (br, ldb) = _rows(g, 1, g.element_size(), H), _rows(beta, 1, beta.element_size(), H)
    with on_device(dev):
        st = _lib.load().ttt_delta_step(qr.data_ptr(), ldq, kr.data_ptr(), ldk, vr.data_ptr(), ldv, gr.data_ptr(), ldg,
                                        br.data_ptr(), ldb, state.data_ptr(), B, H, P, G, N, scale, int(bool(l2_norm)),
                                        *codes, o.data_ptr(), _stream(dev))
    _lib.check(st, "ttt_delta_step")
    torch.autograd.graph.increment_version(state)
    return o


__all__ = ["gated_delta", "gated_delta_step", "GatedDeltaFunction"]
