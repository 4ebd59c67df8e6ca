"""The row loops of the layer norm's and the convolution's backward: more rows than the
workgroups have at once, every number of waves and values to a row, against float64, value by
value."""

import pytest
import torch

from oracle import ssm_oracle as S
from tests import _ssm as T
from tests import _ssm_values as V
from tests.test_gpu_norm import _inputs, _run

pytestmark = pytest.mark.gpu

# D: waves to a row and values to a lane; rows: more than twice what the backward's workgroups
# have at once (four to a workgroup of one-wave rows), and a remainder
NORM = [(200, 6200), (500, 6151), (700, 6213), (1000, 4103),  # one wave: 4, 8, 12, 16 values
        (1025, 1540), (2000, 1601), (2500, 1537), (3500, 1030),  # four: 8, 8, 12, 16
        (5001, 1029), (8000, 515),  # eight: 12, 16
        (10000, 517), (13000, 521), (16384, 513)]  # sixteen: 12, 16, 16


def _norm_reference(d, eps=1e-6):
    """({name: value}, {name: the sum of the absolute values of its terms}) in float64: a row's
    values and their mean over its deviation; backwards the gradient that comes in, its mean
    and its projection on the row."""
    q = {k: None if t is None else t.double() for k, t in d.items()}
    x, z, w, b, dy = (q[k] for k in ("x", "gate", "weight", "bias", "dy"))
    sg = None if z is None else 1 / (1 + torch.exp(-z))
    v = x if z is None else x * z * sg
    u = v - v.mean(-1, keepdim=True)
    rstd = (u.square().mean(-1, keepdim=True) + eps) ** -0.5
    n, g = u * rstd, dy * w
    du = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    ref = {"y": n * w + b, "dx": du if z is None else du * z * sg, "dweight": (dy * n).sum(0), "dbias": dy.sum(0)}
    nm, gm = (v.abs() + v.abs().mean(-1, keepdim=True)) * rstd, g.abs()
    dum = rstd * (gm + gm.mean(-1, keepdim=True) + nm * (gm * nm).mean(-1, keepdim=True))
    size = {"y": nm * w.abs() + b.abs(), "dx": dum if z is None else dum * (z * sg).abs(), "dweight": (dy.abs() * nm).sum(0),
            "dbias": dy.abs().sum(0)}
    if z is not None:
        ref["dgate"] = du * x * sg * (1 + z * (1 - sg))
        size["dgate"] = dum * x.abs() * sg * (1 + z.abs() * (1 - sg))
    return ref, size


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("D,R", NORM)
def test_norm_of_many_rows(lib, dt, D, R, gate):
    parts = lib.ttt_layer_norm_partial_bytes(R, D) // (8 * D)
    assert R > 2 * parts * (4 if D <= 1024 else 1)
    d = T.dev(_inputs(R, D, dt, gate, True, seed=D, pad=3 if D % 2 else 0))
    got = _run(d)
    ref, size = _norm_reference(d)
    assert set(got) == set(ref)
    for k in ref:
        V.each_within(got[k], ref[k], size[k], D + (R if k in ("dweight", "dbias") else 0), f"{k} {(R, D)} {dt}")


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,L,C,W,act,state", [(4200, 30, 130, 4, "silu", True), (11, 7003, 896, 4, "silu", False),
                                               (8300, 31, 40, 3, None, True), (1300, 32, 896, 2, "silu", True)])
def test_conv_of_many_runs(lib, dt, B, L, C, W, act, state):
    """More runs of 32 tokens than the workgroups have at once, and a remainder: the sums of the
    weights' gradients go on over a workgroup's runs."""
    parts = lib.ttt_causal_conv_partial_bytes(B, L, C, W) // (4 * (W + 1) * C)
    assert B * (-(-(L + W - 1) // 32)) > 8 * parts
    d = T.dev(T.conv_inputs(B, L, C, W, dt, seed=C, state=state))
    got = T.conv_run(d, act)
    q = {k: None if t is None else t.double() for k, t in d.items()}
    args = [q[k] for k in T.CONV_ARGS]
    grads = lambda *a, **kw: {"d" + k: v for k, v in S.causal_conv_grads(*args, *a, **kw).items()}  # noqa: E731
    ref, size = grads(act, q["dy"], q["dlast"]), grads(act, q["dy"], q["dlast"], magnitude=True)
    zm = S.causal_conv(*(None if t is None else t.abs() for t in args), None)[0]
    ref["y"], size["y"] = S.causal_conv(*args, act)[0], zm
    if act:  # silu's slope is s (1 + z (1 - s)), at a z that is a sum
        for k, v in grads(None, q["dy"].abs() * (1 + zm), torch.zeros_like(q["dlast"]), magnitude=True).items():
            size[k] = size[k] + v
    for k in got:
        if k != "last":
            V.each_within(got[k], ref[k], size[k], B * L if k in ("dweight", "dbias") else W, f"{k} {(B, L, C)} {dt}")
    s = d["x"] if d["state"] is None else torch.cat([d["state"], d["x"]], 1)
    assert torch.equal(got["last"], s[:, -(W - 1):])  # moved, not computed
