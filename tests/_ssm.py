"""Inputs, references and bounds of the state-space operators' tests."""

from __future__ import annotations

import math

import torch

from oracle import ssm_oracle as S

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SCAN_ARGS = ("x", "dt", "A", "Bm", "Cm", "D", "dt_bias", "state")
CONV_ARGS = ("x", "weight", "bias", "state")


def half_step(dt):
    """The largest relative error of one rounding to dt."""
    return torch.finfo(dt).eps / 2


def within(got, ref, size, terms, what, rounded=None):
    """||got - ref|| against what may separate the two: one rounding to got's own
    type (or to `rounded` as well), and fp32 sums of `terms` terms one after another
    whose absolute values add up to `size`: half a step of the partial sum at each,
    which grow like the root of their number, and half a step for each of the up to
    eight factors of a term (products, exponentials to 1.5 steps, their arguments)."""
    got, ref = got.detach().double().cpu(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    u = 2.0 ** -24
    bound = (half_step(rounded) if rounded is not None else 0.0) * ref.norm() + \
        u * (8 + math.sqrt(terms)) * size.double().norm()
    err = float((got - ref).norm())
    assert err <= float(bound) + 1e-30, f"{what}: off by {err:.3e}, {float(bound):.3e} allowed ({float(ref.norm()):.3e})"


def scan_inputs(B, L, H, P, G, N, dt, seed=0, state=True, skip=True, bias=True, dt_dtype=None, packed=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    if packed:  # columns of one matrix, as the convolution leaves them
        m = r(B, L, H * P + 2 * G * N).to(dt)
        x, b, c = m.split([H * P, G * N, G * N], -1)
        x, b, c = x.unflatten(-1, (H, P)), b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N))
    else:
        x, b, c = r(B, L, H, P).to(dt), r(B, L, G, N).to(dt), r(B, L, G, N).to(dt)
    step = torch.exp(math.log(1e-3) + torch.rand(H, generator=g) * math.log(100.0))
    d = dict(x=x, dt=r(B, L, H).to(dt_dtype or dt), A=-(1 + 15 * torch.rand(H, generator=g)), Bm=b, Cm=c,
             D=r(H) if skip else None, dt_bias=torch.log(torch.expm1(step)) if bias else None,
             state=0.3 * r(B, H, P, N) if state else None)
    d["dy"], d["dlast"] = r(B, L, H, P).to(dt), 0.3 * r(B, H, P, N)
    return d


def dev(d, device="cuda"):
    """The same on the GPU, views still views of one storage where they were."""
    seen = {}
    out = {}
    for k, t in d.items():
        if t is None:
            out[k] = None
            continue
        base = t._base if t._base is not None else t
        if id(base) not in seen:
            seen[id(base)] = base.to(device)
        m = seen[id(base)]
        out[k] = m if base is t else m.as_strided(t.shape, t.stride(), t.storage_offset())
    return out


def scan_reference(d, softplus=True, grads=True):
    """({name: value}, {name: magnitude}) of the outputs and gradients in float64"""
    q = {k: None if t is None else t.double() for k, t in d.items()}
    args = [q[k] for k in SCAN_ARGS]
    ref, size = {}, {}
    ref["y"], ref["last"] = S.selective_scan(*args, softplus=softplus)
    size["y"], size["last"] = S.selective_scan(*args, softplus=softplus, magnitude=True)
    if grads:
        for out, m in ((ref, False), (size, True)):
            out.update({"d" + k: v for k, v in
                        S.selective_scan_grads(*args, softplus, q["dy"], q["dlast"], magnitude=m).items()})
    return ref, size


def scan_run(d, softplus=True, grads=True):
    from ttt_amd.ssm import selective_scan
    leaves = {k: d[k].detach().requires_grad_(grads) for k in SCAN_ARGS if d[k] is not None}
    a = {k: leaves.get(k) for k in SCAN_ARGS}
    y, last = selective_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], a["D"], a["dt_bias"], a["state"],
                             dt_softplus=softplus, return_final_state=True)
    out = {"y": y.detach(), "last": last.detach()}
    if grads:
        gs = torch.autograd.grad([y, last], list(leaves.values()), [d["dy"], d["dlast"]])
        out.update({"d" + k: g for k, g in zip(leaves, gs)})
    return out


def scan_check(d, got, softplus=True, grads=True):
    ref, size = scan_reference(d, softplus, grads)
    B, L, H, P = d["x"].shape
    N = d["Bm"].shape[-1]
    for k in got:
        # the longest sums: over the tokens, a state's row or column, and for the parameters the batch
        terms = L + P + N + (B * L if k in ("dA", "dD", "ddt_bias") else 0)
        dt = got[k].dtype
        within(got[k], ref[k], size[k], terms, f"{k} {tuple(d['x'].shape)} N{N} {d['x'].dtype}",
               rounded=dt if dt != torch.float32 else None)


def conv_inputs(B, L, C, W, dt, seed=0, state=True, bias=True, pad=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(x=r(B, L, C + pad).to(dt)[..., pad:], weight=r(C, W) / W ** 0.5, bias=0.1 * r(C) if bias else None,
                state=r(B, W - 1, C).to(dt) if state else None, dy=r(B, L, C).to(dt), dlast=r(B, W - 1, C).to(dt))


def conv_run(d, act, grads=True):
    from ttt_amd.ssm import causal_conv
    leaves = {k: d[k].detach().requires_grad_(grads) for k in CONV_ARGS if d[k] is not None}
    y, last = causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), leaves.get("state"), act, True)
    out = {"y": y.detach(), "last": last.detach()}
    if grads:
        gs = torch.autograd.grad([y, last], list(leaves.values()), [d["dy"], d["dlast"]])
        out.update({"d" + k: g for k, g in zip(leaves, gs)})
    return out


def conv_check(d, got, act):
    q = {k: None if t is None else t.double() for k, t in d.items()}
    args = [q[k] for k in CONV_ARGS]
    ref, size = {}, {}
    ref["y"], ref["last"] = S.causal_conv(*args, act)
    size["y"], size["last"] = S.causal_conv(*(None if t is None else t.abs() for t in args), None)
    for out, m in ((ref, False), (size, True)):
        out.update({"d" + k: v for k, v in
                    S.causal_conv_grads(*args, act, q["dy"], q["dlast"], magnitude=m).items()})
    B, L, _ = d["x"].shape
    for k in got:
        terms = B * L if k in ("dweight", "dbias") else d["weight"].shape[1]
        dt = got[k].dtype
        within(got[k], ref[k], size[k], terms, f"{k} {tuple(d['x'].shape)} {dt}", dt if dt != torch.float32 else None)
    assert torch.equal(got["last"].cpu(), ref["last"].to(got["last"].dtype))  # moved, not computed
