"""The norms around a block on the GPU against the plain float64 form: widths, types, parts,
layouts by rows and by heads, gradients together and apart, graphs and hooks on saved tensors."""

import math

import pytest
import torch

from oracle import block_oracle as O
from tests import _block as T

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ARGS = ("x", "weight", "residual", "gate", "scale", "next_weight")


def inputs(shape, dt, parts, res_dt=None, seed=0):
    """`parts`: letters of weight, gate, scale, residual and next_weight"""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    D = shape[-1]
    d = dict.fromkeys((*ARGS, "dr", "dy"))
    d["x"] = r(*shape).to(dt)
    if "w" in parts:
        d["weight"] = 1 + 0.1 * r(D)
    if "g" in parts:
        d["gate"] = r(*shape).to(dt)
    if "s" in parts:
        d["scale"] = 0.5 + 0.1 * r(D)
    if "r" in parts:
        d["residual"] = r(*shape).to(res_dt or dt)
    if "n" in parts:
        d["next_weight"] = 1 + 0.1 * r(D)
        d["dy"] = r(*shape).to(dt)
    d["dr"] = r(*shape).to((res_dt or dt) if "r" in parts else dt)
    return d


def run(d, f=None, grads=True):
    if f is None:
        from ttt_amd.norm import block_norm as f
    leaves = {k: d[k].detach().requires_grad_(grads) for k in ARGS if d[k] is not None}
    out = f(*(leaves.get(k) for k in ARGS))
    out = list(out) if isinstance(out, tuple) else [out]
    r = dict(zip(("r", "y"), (t.detach() for t in out)))
    if grads:
        gs = torch.autograd.grad(out, list(leaves.values()), [d["dr"], d["dy"]][:len(out)])
        r.update({"d" + k: t for k, t in zip(leaves, gs)})
    return r


def sizes(d, eps=1e-6):
    """The sums of the absolute values that each result is formed of"""
    x, w, res, z, s, w2, dr, dy = (None if d[k] is None else d[k].double() for k in (*ARGS, "dr", "dy"))
    inv = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5 if w is not None else torch.ones_like(x[..., :1])
    sg = torch.sigmoid(z) if z is not None else None
    gate = (z * sg).abs() if z is not None else 1.0
    dgate = (sg * (1 + z.abs() * (1 - sg))) if z is not None else 0.0
    w1, sc = (1.0 if t is None else t.abs() for t in (w, s))
    u = x.abs() * inv
    m = {"r": u * w1 * gate * sc + (0 if res is None else res.abs())}
    lead = tuple(range(x.dim() - 1))
    D = dr.abs()
    if w2 is not None:
        r = O.block_norm(x, w, res, z, s, None, eps)
        j = ((r * r).mean(-1, keepdim=True) + eps) ** -0.5
        q = m["r"] * j
        m["y"] = q * w2.abs()
        g = dy.abs() * w2.abs()
        D = D + j * (g + q * (g * q).mean(-1, keepdim=True))
        m["dnext_weight"] = (dy.abs() * q).sum(lead)
    m["dresidual"] = D
    m["dscale"] = (D * u * w1 * gate).sum(lead)
    m["dgate"] = D * sc * u * w1 * dgate
    dn = D * sc * gate
    m["dweight"] = (dn * u).sum(lead)
    g = dn * w1 * inv
    m["dx"] = g + u * (g * u).mean(-1, keepdim=True) if w is not None else g
    return m


def check(d, got):
    ref = run({k: None if t is None else t.double() for k, t in d.items()}, O.block_norm)
    size = sizes(d)
    D = d["x"].shape[-1]
    R = d["x"].numel() // D
    for k, t in got.items():
        terms = R if k in ("dweight", "dscale", "dnext_weight") else D
        # (half a step for each of the up to twelve factors of a term, and the sums' partial sums)
        bound = T.U * (12 + math.sqrt(terms)) * size[k].norm()
        if t.dtype != F32:
            bound = bound + T.half_step(t.dtype) * ref[k].norm()
        T.within(t, ref[k], bound, f"{k} {tuple(d['x'].shape)} {d['x'].dtype}")


WIDTHS = [1, 2, 7, 31, 32, 33, 64, 65, 128, 200, 256, 257, 500, 512, 767, 768, 1024, 1025, 2047, 3000, 4096, 4099, 6000, 8192]


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(lib, dt, D):
    for parts, res in (("wg", None), ("wgsrn", F32), ("wsrn", dt)):
        d = inputs((5, D), dt, parts, res, seed=D)
        check(d, run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("parts", ["", "w", "g", "s", "wg", "ws", "wgs", "r", "wr", "sr", "gr", "wgsr", "rn", "wrn", "srn", "grn"])
def test_parts(lib, dt, parts):
    d = inputs((2, 9, 96), dt, parts, F32 if "w" in parts else dt, seed=3)
    check(d, run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R,D", [(1, 768), (5000, 64), (4099, 300), (1700, 1100), (300, 4500)])
def test_many_rows(lib, dt, R, D):
    """More rows than the backward's workgroups have at once."""
    d = inputs((R, D), dt, "wgsrn", F32, seed=R)
    check(d, run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("H,D", [(1, 64), (3, 32), (12, 64), (5, 48), (4, 17)])
def test_heads_of_a_wider_row(lib, dt, H, D):
    """Heads side by side in columns of a projection, and the same from contiguous tensors: the
    same bits, also where one operand has rows of its own."""
    d = T.dev(inputs((2, 7, H, D), dt, "wgsrn", dt, seed=H))
    ref = run(d)
    for wide in (("gate",), ("x", "gate"), ("x", "gate", "residual"), ("residual",)):
        e = dict(d)
        for k in wide:
            m = torch.zeros(2, 7, H * D + 11, device="cuda", dtype=d[k].dtype)
            m[..., 5:5 + H * D] = d[k].flatten(-2)
            e[k] = m[..., 5:5 + H * D].unflatten(-1, (H, D))
        for k, t in run(e).items():
            assert torch.equal(t, ref[k]), (wide, k)
    e = {**d, "x": d["x"].transpose(0, 2).contiguous().transpose(0, 2), "gate": d["gate"].transpose(2, 3).contiguous().transpose(2, 3)}
    for k, t in run(e).items():
        assert torch.equal(t, ref[k]), k
    check({k: None if t is None else t.cpu() for k, t in d.items()}, ref)


def test_gradients_apart(lib):
    """One output's gradient alone, and some inputs' alone."""
    from ttt_amd.norm import block_norm
    d = T.dev(inputs((6, 200), F32, "wgsrn", F32, seed=5))
    full = run(d)
    x = d["x"].detach().requires_grad_(True)
    r, y = block_norm(x, *(d[k] for k in ARGS[1:]))
    (a,) = torch.autograd.grad(r, x, d["dr"], retain_graph=True)
    (b,) = torch.autograd.grad(y, x, d["dy"], retain_graph=True)
    torch.testing.assert_close(a + b, full["dx"], rtol=1e-5, atol=1e-5)
    w = d["weight"].detach().requires_grad_(True)
    r, y = block_norm(d["x"], w, *(d[k] for k in ARGS[2:]))
    (g,) = torch.autograd.grad([r, y], w, [d["dr"], d["dy"]])
    assert torch.equal(g, full["dweight"])
    s = d["scale"].detach().to(BF16).requires_grad_(True)  # a parameter in another type
    (g,) = torch.autograd.grad(block_norm(d["x"], None, None, None, s), s, d["dr"])
    assert g.dtype == BF16


def test_rows_do_not_meet(lib):
    d = T.dev(inputs((9, 130), BF16, "wgsrn", F32, seed=6))
    ref = run(d, grads=False)
    for bad in (math.nan, math.inf):
        e = {**d, "x": d["x"].clone()}
        e["x"][4, 7] = bad
        got = run(e, grads=False)
        keep = [i for i in range(9) if i != 4]
        for k in ref:
            assert torch.equal(got[k][keep], ref[k][keep]) and not torch.isfinite(got[k][4].float()).all()


def test_empty(lib):
    d = T.dev(inputs((0, 3, 64), BF16, "wgsrn", F32))
    got = run(d)
    assert got["r"].shape == (0, 3, 64) and got["r"].dtype == F32 and got["y"].dtype == BF16
    assert (got["dweight"] == 0).all() and (got["dscale"] == 0).all() and (got["dnext_weight"] == 0).all()


def test_in_a_graph_and_on_the_cpu(lib):
    from ttt_amd.norm import block_norm
    d = T.dev(inputs((300, 768), BF16, "wgsrn", F32, seed=7))
    ref = run(d)
    with torch.autograd.graph.save_on_cpu():
        got = run(d)
    for k in ref:
        assert torch.equal(got[k], ref[k]), k
    a = [d[k].clone() for k in ARGS]
    with torch.no_grad():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r, y = block_norm(*a)
        for seed in (8, 9, 10):
            e = T.dev(inputs((300, 768), BF16, "wgsrn", F32, seed=seed))
            for t, k in zip(a, ARGS):
                t.copy_(e[k])
            g.replay()
            wr, wy = block_norm(*a)
            torch.cuda.synchronize()
            assert torch.equal(r, wr) and torch.equal(y, wy)


@pytest.mark.parametrize("parts,res_dt", [("r", BF16), ("r", F32), ("wr", BF16)])
def test_gradient_that_passes_as_it_is(lib, parts, res_dt):
    """The residual's gradient, and a plain x's, may be the result's; the leaves' gradients are each
    its own memory all the same, from one backward to the next."""
    from ttt_amd.norm import block_norm
    d = T.dev(inputs((37, 96), BF16, parts, res_dt, seed=21))
    x, res = (d[k].detach().requires_grad_(True) for k in ("x", "residual"))
    dr = d["dr"].clone()
    for n in (1, 2):
        block_norm(x, d["weight"], res).backward(dr)
        assert torch.equal(dr, d["dr"]) and torch.equal(res.grad, n * dr)
        if parts == "r":
            assert torch.equal(x.grad, n * dr.to(BF16))
    assert len({x.grad.data_ptr(), res.grad.data_ptr(), dr.data_ptr()}) == 3
    x.grad.zero_()
    assert torch.equal(res.grad, 2 * dr) and torch.equal(dr, d["dr"])
