"""Layer norm over the last axis, plain and gated, against the plain float64 form."""

import pytest
import torch

from oracle import ssm_oracle as S
from tests import _ssm as T

pytestmark = pytest.mark.gpu


def _inputs(R, D, dt, gate, affine, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(x=r(R, D + pad).to(dt)[:, pad:], gate=r(R, D).to(dt) if gate else None,
                weight=1 + 0.1 * r(D) if affine else None, bias=r(D) if affine else None, dy=r(R, D).to(dt))


def _run(d):
    from ttt_amd.norm import layer_norm
    leaves = {k: d[k].detach().requires_grad_(True) for k in ("x", "gate", "weight", "bias") if d[k] is not None}
    y = layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), leaves.get("gate"))
    gs = torch.autograd.grad(y, list(leaves.values()), d["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, gs)}}


def _check(d, got, eps=1e-6):
    q = {k: None if t is None else t.double() for k, t in d.items()}
    leaves = {k: q[k].requires_grad_(True) for k in ("x", "gate", "weight", "bias") if q[k] is not None}
    y = S.layer_norm(q["x"], q["weight"], q["bias"], q["gate"], eps)
    gs = torch.autograd.grad(y, list(leaves.values()), q["dy"])
    ref = {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, gs)}}
    # what the values are sums of: a row's values over its own deviation, and in the
    # backward the incoming gradient, its mean and its projection on the row
    with torch.no_grad():
        sil = 1.0 if q["gate"] is None else (q["gate"] * torch.sigmoid(q["gate"])).abs()
        dsil = None if q["gate"] is None else (torch.sigmoid(q["gate"]) * (1 + q["gate"] * (1 - torch.sigmoid(q["gate"])))).abs()
        v = q["x"].abs() * sil
        rstd = (v if q["gate"] is None else v)
        u = q["x"] * (1.0 if q["gate"] is None else q["gate"] * torch.sigmoid(q["gate"]))
        rstd = ((u - u.mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + eps) ** -0.5
        n = (v + v.mean(-1, keepdim=True)) * rstd
        w = 1.0 if q["weight"] is None else q["weight"].abs()
        dn = q["dy"].abs() * w
        du = rstd * (dn + dn.mean(-1, keepdim=True) + n * (dn * n).mean(-1, keepdim=True))
        size = {"y": n * w + (0 if q["bias"] is None else q["bias"].abs()), "dx": du * sil,
                "dweight": (q["dy"].abs() * n).sum(0), "dbias": q["dy"].abs().sum(0)}
        if dsil is not None:
            size["dgate"] = du * q["x"].abs() * dsil
    R, D = d["x"].shape
    for k in got:
        dt = got[k].dtype
        T.within(got[k], ref[k], size[k], R if k in ("dweight", "dbias") else D, f"{k} {(R, D)} {dt}",
                 None if dt == torch.float32 else dt)


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R,D,gate,affine,pad", [
    (1, 1, False, True, 0), (1, 2, True, True, 0), (3, 7, False, False, 0), (5, 8, True, True, 8), (9, 64, False, True, 0),
    (4, 511, True, True, 1), (1031, 512, False, True, 0), (6, 513, False, True, 3), (70, 768, True, True, 24),
    (3, 1024, True, False, 0), (2, 1025, False, True, 0), (300, 2047, True, True, 1), (5, 2048, False, True, 0),
    (4, 4097, True, True, 0), (2, 8193, True, True, 0), (2, 16384, True, True, 0), (3, 16383, False, True, 5)])
def test_layer_norm(lib, dt, R, D, gate, affine, pad):
    d = _inputs(R, D, dt, gate, affine, seed=R + D, pad=pad)
    _check(d, _run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_rows_far_from_zero(lib, dt):
    """A mean far above the deviation: the variance is that of the centred values."""
    d = _inputs(6, 300, dt, False, True, seed=3)
    d["x"] = (d["x"].float() + 60.0).to(dt)
    _check(d, _run(T.dev(d)))


def test_constant_rows(lib):
    """Rows without a deviation: the bias, and a finite gradient."""
    d = _inputs(4, 96, torch.float32, False, True, seed=4)
    d["x"] = torch.full((4, 96), 3.0)
    got = _run(T.dev(d))
    assert torch.equal(got["y"].cpu(), d["bias"].expand(4, 96))
    assert torch.isfinite(got["dx"]).all()


def test_leading_axes_and_layouts(lib):
    from ttt_amd.norm import layer_norm
    x = torch.randn(3, 5, 7, 40, device="cuda").to(torch.bfloat16)
    w, b = torch.randn(40, device="cuda"), torch.randn(40, device="cuda")
    want = layer_norm(x.reshape(-1, 40), w, b).view(3, 5, 7, 40)
    assert torch.equal(layer_norm(x, w, b), want)
    assert torch.equal(layer_norm(x.transpose(0, 2), w, b), want.transpose(0, 2))
    assert torch.equal(layer_norm(x[0, 0, 0], w, b), want[0, 0, 0])
    wide = torch.randn(3, 5, 7, 90, device="cuda").to(torch.bfloat16)
    wide[..., 11:51] = x
    assert torch.equal(layer_norm(wide[..., 11:51], w, b), want)
    e = x[0, 0, :1].expand(7, 40)
    assert torch.equal(layer_norm(e, w, b), want[0, 0, :1].expand(7, 40))


def test_rows_that_are_not_finite_stay_alone(lib):
    from ttt_amd.norm import layer_norm
    x = torch.randn(9, 200, device="cuda")
    want = layer_norm(x)
    x[4, 3] = float("nan")
    got = layer_norm(x)
    keep = torch.arange(9, device="cuda") != 4
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[4]).all()


def test_repeats_and_graph(lib):
    d = T.dev(_inputs(500, 768, torch.bfloat16, True, True, seed=5))
    a, b = _run(d), _run(d)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _run(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(d)
    for seed in (6, 7, 8):
        new = T.dev(_inputs(500, 768, torch.bfloat16, True, True, seed=seed))
        for k, t in new.items():
            d[k].copy_(t)
        want = _run(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(out[k], want[k]), (seed, k)
