"""The selective state-space operators in plain PyTorch, from their definitions and
token by token: what the kernels are tested against, on the CPU in float64.

`magnitude=True` gives, instead of a gradient, the sum of the absolute values of
the terms that it is a sum of: what the rounding errors of any order of summation
are proportional to.  (Decays are positive either way.)"""

from __future__ import annotations

import torch


def _silu(z):
    return z / (1 + torch.exp(-z))


def _dsilu(z):
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def causal_conv(x, weight, bias=None, state=None, activation=None):
    """(y [B,L,C], the last W-1 inputs)"""
    B, L, C = x.shape
    W = weight.shape[1]
    s = torch.cat([x.new_zeros(B, W - 1, C) if state is None else state, x], 1)
    z = x.new_zeros(B, L, C) + (0 if bias is None else bias)
    for k in range(W):
        z = z + weight[:, k] * s[:, k:k + L]
    return _silu(z) if activation == "silu" else z, s[:, L:]


def causal_conv_grads(x, weight, bias, state, activation, dy, dlast, magnitude=False):
    """{"x", "weight", "bias", "state"}: gradients of sum(y dy) + sum(last dlast)"""
    B, L, C = x.shape
    W = weight.shape[1]
    s = torch.cat([x.new_zeros(B, W - 1, C) if state is None else state, x], 1)
    z = x.new_zeros(B, L, C) + (0 if bias is None else bias)
    for k in range(W):
        z = z + weight[:, k] * s[:, k:k + L]
    f = _dsilu(z) if activation == "silu" else torch.ones_like(z)
    if magnitude:
        s, weight, dy, dlast, f = s.abs(), weight.abs(), dy.abs(), dlast.abs(), f.abs()
    dz = dy * f
    ds, dw = torch.zeros_like(s), torch.zeros_like(weight)
    ds[:, L:] += dlast
    for k in range(W):
        ds[:, k:k + L] += weight[:, k] * dz
        dw[:, k] = (dz * s[:, k:k + L]).sum((0, 1))
    return {"x": ds[:, W - 1:], "weight": dw, "bias": dz.sum((0, 1)), "state": ds[:, :W - 1]}


def _steps(dt, dt_bias, softplus):
    raw = dt if dt_bias is None else dt + dt_bias
    if not softplus:
        return raw, raw, torch.ones_like(raw)
    return raw, torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())), 1 / (1 + torch.exp(-raw))


def selective_scan(x, dt, A, Bm, Cm, D=None, dt_bias=None, h0=None, softplus=True, magnitude=False):
    """(y [B,L,H,P], the last state [B,H,P,N])"""
    B, L, H, P = x.shape
    rep, N = H // Bm.shape[2], Bm.shape[3]
    d = _steps(dt, dt_bias, softplus)[1]
    a = torch.exp(d * A)
    b, c = Bm.repeat_interleave(rep, 2), Cm.repeat_interleave(rep, 2)
    h = x.new_zeros(B, H, P, N) if h0 is None else h0
    if magnitude:
        x, b, c, h, D = x.abs(), b.abs(), c.abs(), h.abs(), None if D is None else D.abs()
    y = []
    for t in range(L):
        h = a[:, t, :, None, None] * h + (d[:, t, :, None] * x[:, t])[..., None] * b[:, t, :, None, :]
        y.append((h * c[:, t, :, None, :]).sum(-1) + (0 if D is None else D[:, None] * x[:, t]))
    return torch.stack(y, 1), h


def selective_scan_grads(x, dt, A, Bm, Cm, D, dt_bias, h0, softplus, dy, dlast, magnitude=False):
    """{"x", "dt", "A", "Bm", "Cm", "D", "dt_bias", "state"}: gradients of
    sum(y dy) + sum(last dlast), walked back from the last token"""
    B, L, H, P = x.shape
    G, N = Bm.shape[2:]
    rep = H // G
    raw, d, ds = _steps(dt, dt_bias, softplus)
    a = torch.exp(d * A)
    b, c = Bm.repeat_interleave(rep, 2), Cm.repeat_interleave(rep, 2)
    h = x.new_zeros(B, H, P, N) if h0 is None else h0
    skip = torch.zeros_like(A) if D is None else D
    rate = A
    if magnitude:
        x, b, c, h, skip, dy, dlast, rate = (t.abs() for t in (x, b, c, h, skip, dy, dlast, rate))
    before = []
    for t in range(L):
        before.append(h)
        h = a[:, t, :, None, None] * h + (d[:, t, :, None] * x[:, t])[..., None] * b[:, t, :, None, :]
    g = dlast.clone()
    dx, dd, db, dc = torch.zeros_like(x), torch.zeros_like(d), torch.zeros_like(b), torch.zeros_like(c)
    dA = torch.zeros_like(A)
    for t in reversed(range(L)):
        dc[:, t] = (dy[:, t, :, :, None] * h).sum(2)
        g = g + dy[:, t, :, :, None] * c[:, t, :, None, :]
        h = before[t]
        gb = (g * b[:, t, :, None, :]).sum(-1)
        da = a[:, t] * (g * h).sum((-1, -2))
        dx[:, t] = d[:, t, :, None] * gb + skip[:, None] * dy[:, t]
        db[:, t] = d[:, t, :, None] * (g * x[:, t, :, :, None]).sum(2)
        dd[:, t] = (gb * x[:, t]).sum(-1) + rate * da
        dA += (da * d[:, t]).sum(0)
        g = a[:, t, :, None, None] * g
    ddt = dd * ds
    return {"x": dx, "dt": ddt, "A": dA, "Bm": db.unflatten(2, (G, rep)).sum(3), "Cm": dc.unflatten(2, (G, rep)).sum(3),
            "D": (dy * x).sum((0, 1, 3)), "dt_bias": ddt.sum((0, 1)), "state": g}


def layer_norm(x, weight=None, bias=None, gate=None, eps=1e-6):
    v = x if gate is None else x * _silu(gate)
    u = v - v.mean(-1, keepdim=True)
    n = u / torch.sqrt((u * u).mean(-1, keepdim=True) + eps)
    return n if weight is None else n * weight + bias
