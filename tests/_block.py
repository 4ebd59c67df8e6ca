"""Inputs, references and bounds of the tests of a gated delta-rule block's operators."""

from __future__ import annotations

import math

import torch

from oracle import block_oracle as O
from tests._ssm import dev, half_step  # noqa: F401

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DELTA_ARGS = ("q", "k", "v", "g", "beta", "state")
U = 2.0 ** -24


def within(got, ref, bound, what):
    """||got - ref|| <= bound, a number in the 2-norm over the whole tensor"""
    got, ref = got.detach().double().cpu(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    err = float((got - ref).norm())
    assert err <= float(bound) + 1e-30, f"{what}: off by {err:.3e}, {float(bound):.3e} allowed ({float(ref.norm()):.3e})"


def delta_inputs(B, L, H, G, N, P, dt, seed=0, state=True, unit=True, packed=True, g_dtype=torch.float32,
                 beta_dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    z = r(B, L, 2 * G * N + H * P)
    z = z / (1 + torch.exp(-z))
    if not unit:
        z[..., :2 * G * N] = O._unit(z[..., :2 * G * N].unflatten(-1, (2 * G, N))).flatten(-2)
    z = z.to(dt)
    q, k, v = z.split([G * N, G * N, H * P], -1)
    q, k, v = q.unflatten(-1, (G, N)), k.unflatten(-1, (G, N)), v.unflatten(-1, (H, P))
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    step = torch.exp(math.log(1e-3) + torch.rand(H, generator=gen) * math.log(100.0))
    a = r(B, L, H) + torch.log(torch.expm1(step))
    d = dict(q=q, k=k, v=v, g=(-(1 + 15 * torch.rand(H, generator=gen)) * torch.log1p(torch.exp(a))).to(g_dtype),
             beta=torch.sigmoid(r(B, L, H)).to(beta_dtype), state=0.3 * r(B, H, P, N) if state else None)
    d["do"], d["dlast"] = r(B, L, H, P).to(dt), 0.3 * r(B, H, P, N)
    return d


def delta_run(d, unit=True, scale=None, grads=True):
    from ttt_amd.delta import gated_delta
    leaves = {k: d[k].detach().requires_grad_(grads) for k in DELTA_ARGS if d[k] is not None}
    a = {k: leaves.get(k) for k in DELTA_ARGS}
    o, last = gated_delta(a["q"], a["k"], a["v"], a["g"], a["beta"], a["state"], scale, unit, True)
    out = {"o": o.detach(), "last": last.detach()}
    if grads:
        gs = torch.autograd.grad([o, last], list(leaves.values()), [d["do"], d["dlast"]])
        out.update({"d" + k: t for k, t in zip(leaves, gs)})
    return out


def delta_check(d, got, unit=True, scale=None):
    """Against the definition in float64.  A result may be off by one rounding to its own type; by
    what forming it gives, half a step for each of the up to eight factors of a term and for the
    partial sums of its N + P terms, which grow like the root of their number; and by as much for
    each token that the state went through: a token's update, of norm 1 or less (keys of unit
    length or less, weights up to 1), carries the errors made before it and enlarges none, and
    errors of L tokens add up like the root of L.  In bf16 calls, results of that type take two
    factors rounded to 2^-17."""
    q = {k: None if t is None else t.double() for k, t in d.items()}
    args = [q[k] for k in ("q", "k", "v", "g", "beta", "state", "do", "dlast")]
    ref, size = (O.gated_delta_all(*args, scale=scale, unit=unit, sizes=s) for s in (False, True))
    B, L, H, P = d["v"].shape
    N = d["k"].shape[-1]
    act = d["v"].dtype
    for k, t in got.items():
        bound = U * (8 + math.sqrt(N + P)) * (1 + math.sqrt(L)) * size[k].norm()
        if t.dtype != torch.float32:
            bound = bound + half_step(t.dtype) * ref[k].norm()
        if act == torch.bfloat16 and t.dtype == act:
            bound = bound + 2 * 2.0 ** -17 * size[k].norm()
        within(t, ref[k], bound, f"{k} {tuple(d['v'].shape)} N{N} {act}")
