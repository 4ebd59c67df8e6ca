"""A gated delta-rule block's operators in plain PyTorch, from their definitions: what the
kernels are tested against, on the CPU in float64.

`sizes=True` gives, in place of a value, the sum of the absolute values of the terms that
it is a sum of, taken with the exact values of what was formed before it: what the rounding
errors made in forming it are proportional to."""

from __future__ import annotations

import math

import torch

UNIT_EPS = 1e-6


def _unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + UNIT_EPS)


def gated_delta(q, k, v, g, beta, h0=None, scale=None, unit=True):
    """(o [B,L,H,P], the last state [B,H,P,N]), token by token"""
    B, L, H, P = v.shape
    G, N = k.shape[2:]
    scale = N ** -0.5 if scale is None else scale
    q, k = (_unit(t) if unit else t for t in (q, k))
    q, k = (t.repeat_interleave(H // G, 2)[:, :, :, None] for t in (q, k))  # [B,L,H,1,N]
    s = v.new_zeros(B, H, P, N) if h0 is None else h0
    o = []
    for t in range(L):
        s = s * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (s * k[:, t]).sum(-1))
        s = s + u[..., None] * k[:, t]
        o.append(scale * (s * q[:, t]).sum(-1))
    return (torch.stack(o, 1) if L else v.new_zeros(B, 0, H, P)), s


def gated_delta_all(q, k, v, g, beta, h0, do, dlast, scale=None, unit=True, sizes=False):
    """{"o", "last", "dq", "dk", "dv", "dg", "dbeta", "dstate"}: the values and the gradients of
    sum(o do) + sum(last dlast), walked back from the last token"""
    B, L, H, P = v.shape
    G, N = k.shape[2:]
    scale = N ** -0.5 if scale is None else scale
    m = (lambda t: t.abs()) if sizes else (lambda t: t)
    rq, rk = ((t.square().sum(-1, keepdim=True) + UNIT_EPS) ** -0.5 if unit else torch.ones_like(t[..., :1]) for t in (q, k))
    qu, ku = q * rq, k * rk
    qh, kh = (t.repeat_interleave(H // G, 2)[:, :, :, None] for t in (qu, ku))
    s = v.new_zeros(B, H, P, N) if h0 is None else h0
    before, miss, os, size = [], [], [], None
    a = torch.exp(g)
    for t in range(L):
        before.append(s)
        old = s * a[:, t, :, None, None]
        x = v[:, t] - (old * kh[:, t]).sum(-1)
        miss.append(x)
        u = beta[:, t, :, None] * x
        s = old + u[..., None] * kh[:, t]
        os.append((m(s) * m(qh[:, t])).sum(-1) * scale)
        if sizes:
            size = m(old) + (beta[:, t, :, None].abs() * (m(v[:, t]) + (m(old) * m(kh[:, t])).sum(-1)))[..., None] * m(kh[:, t])
    r = {"o": torch.stack(os, 1), "last": size if sizes else s}
    ds = dlast.clone()
    dqh, dkh, dv = torch.empty(B, L, H, N, dtype=v.dtype), torch.empty(B, L, H, N, dtype=v.dtype), torch.empty_like(v)
    dg, db = torch.empty_like(g), torch.empty_like(beta)
    dsize = m(ds)
    for t in reversed(range(L)):
        do_t = scale * do[:, t, ..., None]
        dqh[:, t] = (m(do_t) * m(s)).sum(2)
        ds = ds + do_t * qh[:, t]
        dsize = m(ds) if sizes else None
        s, x, kt, bt = before[t], miss[t], kh[:, t], beta[:, t, :, None]
        old = s * a[:, t, :, None, None]
        du = (ds * kt).sum(-1)
        dr = bt * du
        dv[:, t] = m(bt) * (m(ds) * m(kt)).sum(-1)
        db[:, t] = ((m(ds) * m(kt)).sum(-1) * m(x)).sum(-1)
        dkh[:, t] = (m(ds) * m(bt * x)[..., None]).sum(2) + (1 if sizes else -1) * (m(dr)[..., None] * m(old)).sum(2)
        dold = ds - dr[..., None] * kt
        dg[:, t] = ((m(ds) + m(dr)[..., None] * m(kt)) * m(old)).sum((-1, -2)) if sizes else (dold * old).sum((-1, -2))
        ds = dold * a[:, t, :, None, None]
    if sizes:
        ds = ds.abs() + (dsize * a[:, 0, :, None, None] if L else 0)
    dq, dk = (t.unflatten(2, (G, H // G)).sum(3) for t in (dqh, dkh))
    if unit:
        sign = 1 if sizes else -1
        dq, dk = (rr * (d + sign * m(y) * (m(d) * m(y)).sum(-1, keepdim=True)) for rr, d, y in ((rq, dq, qu), (rk, dk, ku)))
    r.update(dq=dq, dk=dk, dv=dv, dg=dg, dbeta=db, dstate=ds)
    return r


def block_norm(x, weight=None, residual=None, gate=None, scale=None, next_weight=None, eps=1e-6):
    n = x if weight is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    if gate is not None:
        n = n * gate / (1 + torch.exp(-gate))
    if scale is not None:
        n = n * scale
    if residual is None:
        return n
    r = residual + n
    return r if next_weight is None else (r, r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * next_weight)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    a, b = x @ w_gate.T, x @ w_up.T
    a = a if b_gate is None else a + b_gate
    b = b if b_up is None else b + b_up
    f = a / (1 + torch.exp(-a)) if activation == "silu" else 0.5 * a * torch.erfc(-a / math.sqrt(2.0))
    return f * b
