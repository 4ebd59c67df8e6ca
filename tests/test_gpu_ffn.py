"""The gated feed-forward projections on the GPU against the plain float64 form: sizes on both
sides of every tile, types, activations, biases, layouts, gradients together and apart, graphs."""

import math

import pytest
import torch

from oracle import block_oracle as O
from tests import _block as T

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ARGS = ("x", "w_gate", "w_up", "b_gate", "b_up")


def inputs(R, D, F, dt, bias=True, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(x=r(R, D + pad).to(dt)[:, :D], w_gate=(r(F, D) / D ** 0.5).to(dt), w_up=(r(F, D) / D ** 0.5).to(dt),
                b_gate=(0.3 * r(F)).to(dt) if bias else None, b_up=(0.3 * r(F)).to(dt) if bias else None,
                dy=r(R, F).to(dt))


def run(d, act="silu", grads=True):
    from ttt_amd.ffn import gated_linear
    leaves = {k: d[k].detach().requires_grad_(grads) for k in ARGS if d[k] is not None}
    y = gated_linear(*(leaves.get(k) for k in ARGS), activation=act)
    out = {"y": y.detach()}
    if grads:
        out.update({"d" + k: t for k, t in zip(leaves, torch.autograd.grad(y, list(leaves.values()), d["dy"]))})
    return out


def check(d, got, act="silu"):
    """A result may be off by one rounding to its type, by the rounding errors of fp32 sums of D, F
    or R terms, and the gradients that the 16-bit calls round to their type by those roundings:
    half a step of each term at most, whose signs have nothing to do with one another."""
    q = {k: None if t is None else t.double() for k, t in d.items()}
    x, wg, wu, dy = q["x"], q["w_gate"], q["w_up"], q["dy"]
    a, b, sa, sb = x @ wg.T, x @ wu.T, x.abs() @ wg.abs().T, x.abs() @ wu.abs().T
    if q["b_gate"] is not None:
        a, b, sa, sb = a + q["b_gate"], b + q["b_up"], sa + q["b_gate"].abs(), sb + q["b_up"].abs()
    if act == "silu":
        s = torch.sigmoid(a)
        f, df, ddf = a * s, s * (1 + a * (1 - s)), 0.5
    else:
        s = 0.5 * torch.erfc(-a / math.sqrt(2))
        f, df, ddf = a * s, s + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi), 0.8
    da, db = dy * b * df, dy * f
    (R, D), F = x.shape, wg.shape[0]
    u = lambda n: T.U * (8 + math.sqrt(n))  # noqa: E731
    # what a and b are off by reaches the rest through the derivatives (|f'| <= 1.13, |f''| <= ddf)
    ea, eb = u(D) * sa, u(D) * sb
    ey = 1.13 * ea * b.abs() + f.abs() * eb + 8 * T.U * (f * b).abs()
    eda = dy.abs() * (eb * df.abs() + b.abs() * ddf * ea) + 8 * T.U * da.abs()
    edb = dy.abs() * 1.13 * ea + 8 * T.U * db.abs()
    h = T.half_step(d["x"].dtype) if d["x"].dtype != F32 else 0.0
    sq = lambda t: t.square()  # noqa: E731
    ref = {"y": f * b, "dx": da @ wg + db @ wu, "dw_gate": da.T @ x, "dw_up": db.T @ x, "db_gate": da.sum(0), "db_up": db.sum(0)}
    err = {"y": ey,
           "dx": eda @ wg.abs() + edb @ wu.abs() + u(2 * F) * (da.abs() @ wg.abs() + db.abs() @ wu.abs())
           + h * torch.sqrt(sq(da) @ sq(wg) + sq(db) @ sq(wu)),
           "dw_gate": eda.T @ x.abs() + u(R) * (da.abs().T @ x.abs()) + h * torch.sqrt(sq(da).T @ sq(x)),
           "dw_up": edb.T @ x.abs() + u(R) * (db.abs().T @ x.abs()) + h * torch.sqrt(sq(db).T @ sq(x)),
           "db_gate": eda.sum(0) + u(R) * da.abs().sum(0), "db_up": edb.sum(0) + u(R) * db.abs().sum(0)}
    for k, t in got.items():
        T.within(t, ref[k], err[k].norm() + h * ref[k].norm(), f"{k} {R}x{D}x{F} {d['x'].dtype} {act}")


SHAPES = [(1, 1, 1), (1, 8, 16), (2, 7, 3), (16, 32, 16), (17, 33, 15), (31, 64, 100), (33, 100, 65), (64, 256, 40),
          (65, 24, 17), (100, 129, 64), (128, 64, 64), (129, 65, 66), (255, 40, 200), (300, 136, 72), (700, 16, 8), (513, 200, 333)]


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R,D,F", SHAPES)
def test_sizes(lib, dt, R, D, F):
    d = inputs(R, D, F, dt, bias=R % 2 == 1, seed=R + D + F)
    act = "gelu" if F % 2 else "silu"
    check(d, run(T.dev(d), act), act)


@pytest.mark.parametrize("dt,R,D,F", [(BF16, 6200, 72, 1100), (F16, 6200, 40, 1030), (F32, 6200, 24, 1030)])
def test_large_tiles(lib, dt, R, D, F):
    """Enough tiles of 256 x 256, for dW in shares of the rows."""
    d = inputs(R, D, F, dt, seed=1)
    check(d, run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_one_bias(lib, dt):
    from ttt_amd.ffn import gated_linear
    d = T.dev(inputs(70, 40, 50, dt, seed=2))
    z = torch.zeros_like(d["b_up"])
    for R in (70, 9):
        x = d["x"][:R]
        assert torch.equal(gated_linear(x, d["w_gate"], d["w_up"], d["b_gate"]),
                           gated_linear(x, d["w_gate"], d["w_up"], d["b_gate"], z))
        assert torch.equal(gated_linear(x, d["w_gate"], d["w_up"], None, d["b_up"]),
                           gated_linear(x, d["w_gate"], d["w_up"], z, d["b_up"]))
    b = d["b_gate"].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(gated_linear(d["x"], d["w_gate"], d["w_up"], b, d["b_up"]), b, d["dy"])
    assert torch.equal(g, run(d)["db_gate"])


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R", [5, 90])
def test_layouts(lib, dt, R):
    """x as columns of a wider matrix, off 16 bytes, transposed; weights off 16 bytes; leading axes:
    the same bits."""
    from ttt_amd.ffn import gated_linear
    d = T.dev(inputs(R, 48, 40, dt, seed=3))
    ref = run(d)
    for pad, first in ((8, 0), (8, 8), (3, 1), (3, 2)):
        m = torch.zeros(R, 48 + pad, device="cuda", dtype=dt)
        m[:, first:first + 48] = d["x"]
        for k, t in run({**d, "x": m[:, first:first + 48]}).items():
            assert torch.equal(t, ref[k]), (pad, first, k)
    w = torch.zeros(40 * 48 + 1, device="cuda", dtype=dt)
    w[1:] = d["w_gate"].flatten()
    e = {**d, "x": d["x"].t().contiguous().t(), "w_gate": w[1:].view(40, 48), "w_up": d["w_up"].t().contiguous().t(),
         "dy": d["dy"].t().contiguous().t()}
    for k, t in run(e).items():
        assert torch.equal(t, ref[k]), k
    y = gated_linear(d["x"].view(R // 5, 5, 48), *(d[k] for k in ARGS[1:]))
    assert torch.equal(y.view(R, 40), ref["y"])


def test_gradients_apart(lib):
    from ttt_amd.ffn import gated_linear
    d = T.dev(inputs(90, 48, 40, F32, seed=4))
    full = run(d)
    for k in ARGS:
        a = {q: d[q] for q in ARGS}
        a[k] = d[k].detach().requires_grad_(True)
        (g,) = torch.autograd.grad(gated_linear(*a.values()), a[k], d["dy"])
        assert torch.equal(g, full["d" + k]), k


@pytest.mark.parametrize("R", [9, 90])
def test_rows_do_not_meet(lib, R):
    d = T.dev(inputs(R, 100, 60, BF16, seed=5))
    ref = run(d, grads=False)["y"]
    for bad in (math.nan, math.inf):
        e = {**d, "x": d["x"].clone()}
        e["x"][4, 99] = bad
        got = run(e, grads=False)["y"]
        keep = [i for i in range(R) if i != 4]
        assert torch.equal(got[keep], ref[keep]) and not torch.isfinite(got[4].float()).any()


def test_empty(lib):
    d = T.dev(inputs(0, 48, 40, BF16))
    got = run(d)
    assert got["y"].shape == (0, 40) and got["dx"].shape == (0, 48) and (got["dw_gate"] == 0).all()


def test_in_a_graph_and_on_the_cpu(lib):
    from ttt_amd.ffn import gated_linear
    for dt, R in ((BF16, 300), (F32, 300), (BF16, 3)):
        d = T.dev(inputs(R, 96, 72, dt, seed=6))
        ref = run(d)
        with torch.autograd.graph.save_on_cpu():
            got = run(d)
        for k in ref:
            assert torch.equal(got[k], ref[k]), k
        a = [d[k].clone() for k in ARGS]
        with torch.no_grad():
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = gated_linear(*a)
            for seed in (7, 8, 9):
                e = T.dev(inputs(R, 96, 72, dt, seed=seed))
                for t, k in zip(a, ARGS):
                    t.copy_(e[k])
                g.replay()
                want = gated_linear(*a)
                torch.cuda.synchronize()
                assert torch.equal(y, want)


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R,D,F,bias", [(4099, 400, 2100, False), (4099, 4200, 200, True)])
def test_rounds_of_large_tiles_and_what_is_left(lib, dt, R, D, F, bias):
    """More than a round of large tiles and less than two, of both projections' columns and of dx:
    what is left of them is cut in four."""
    d = inputs(R, D, F, dt, bias=bias, seed=R + D)
    check(d, run(T.dev(d)))
