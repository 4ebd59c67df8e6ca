"""The gated delta rule on the GPU against the plain float64 form, over sizes, types, layouts
and states; a prompt in parts and token by token; weights and decays at their ends; values
that are not finite; graphs, streams, hooks on saved tensors and repeated calls."""

import math

import pytest
import torch

from oracle import block_oracle as O
from tests import _block as T

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

SHAPES = [  # B, L, H, G, N, P
    (1, 1, 1, 1, 16, 32), (2, 2, 2, 1, 64, 64), (1, 15, 3, 3, 48, 32), (2, 16, 2, 2, 32, 64), (1, 17, 4, 2, 128, 64),
    (1, 31, 2, 1, 64, 96), (2, 33, 1, 1, 80, 128), (3, 63, 6, 3, 64, 32), (1, 65, 2, 2, 16, 256), (2, 129, 4, 1, 96, 64),
    (1, 200, 3, 3, 128, 128), (2, 333, 2, 2, 64, 64)]


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,L,H,G,N,P", SHAPES)
def test_delta(lib, dt, B, L, H, G, N, P):
    d = T.delta_inputs(B, L, H, G, N, P, dt, seed=B + L + N)
    T.delta_check(d, T.delta_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("state,unit,scale,g32,b32", [
    (False, False, None, True, False), (True, False, 0.7, False, True), (False, True, 1.0, False, False)])
def test_options(lib, dt, state, unit, scale, g32, b32):
    d = T.delta_inputs(2, 70, 4, 2, 64, 64, dt, seed=5, state=state, unit=unit, g_dtype=F32 if g32 else dt,
                       beta_dtype=F32 if b32 else dt)
    T.delta_check(d, T.delta_run(T.dev(d), unit, scale), unit, scale)


@pytest.mark.parametrize("dt,L", [(BF16, 1500), (F32, 700), (F16, 900)])
def test_long_single_sequence(lib, dt, L):
    """Few chains: the length is cut into many segments."""
    d = T.delta_inputs(1, L, 1, 1, 32, 32, dt, seed=9)
    T.delta_check(d, T.delta_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("N,P", [(16, 64), (32, 128), (32, 96), (48, 64), (128, 64), (96, 32)])
def test_segments_of_each_width(lib, dt, N, P):
    """The segments' products, of every width of the state, with more and fewer columns than a
    workgroup has."""
    d = T.delta_inputs(1, 1100, 2, 1, N, P, dt, seed=N + P)
    T.delta_check(d, T.delta_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_many_chains(lib, dt):
    """More sequences and heads than workgroups are held at once: one segment of each."""
    d = T.delta_inputs(70, 70, 8, 4, 16, 32, dt, seed=10)
    T.delta_check(d, T.delta_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_weights_and_decays_at_their_ends(lib, dt):
    """Weights of 0 (nothing is written) and 1, decays of 0, of e^-600 and less and of nothing
    left (g = -inf), next to one another; keys that repeat, so that a chunk's system has
    entries of 1."""
    d = T.delta_inputs(2, 150, 3, 3, 32, 64, dt, seed=6)
    d["beta"][:, 3::7] = 0.0
    d["beta"][:, 5::11] = 1.0
    d["g"][:, ::5] = 0.0
    d["g"][:, 10::23] = -600.0
    d["g"][:, 17::41] = -math.inf
    d["k"] = d["k"].clone()
    d["k"][:, 40:60] = d["k"][:, 40:41]
    ref = {**d, "g": d["g"].clamp(min=-1e4)}
    got = T.delta_run(T.dev(d))
    T.delta_check(ref, got)
    assert (got["dv"].cpu()[d["beta"] == 0] == 0).all()  # (some of those set to 0 were set to 1 after)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_layouts(lib, dt):
    """Columns of one matrix, contiguous tensors, rows off 16 bytes and transposed memory give
    the same bits."""
    d = T.dev(T.delta_inputs(2, 75, 4, 2, 64, 64, dt, seed=7))
    ref = T.delta_run(d)
    for how in ("contiguous", "odd rows", "transposed"):
        e = dict(d)
        for k in ("q", "k", "v", "g", "beta"):
            t = d[k]
            if how == "contiguous":
                e[k] = t.contiguous()
            elif how == "odd rows":
                flat = t.flatten(2)
                m = torch.zeros(2, 75, flat.shape[2] + 3, device="cuda", dtype=t.dtype)
                m[..., 1:-2] = flat
                e[k] = m[..., 1:-2].unflatten(2, t.shape[2:])
            else:
                e[k] = t.transpose(0, 1).contiguous().transpose(0, 1)
        e["do"] = d["do"].transpose(0, 1).contiguous().transpose(0, 1) if how == "transposed" else d["do"]
        for k, t in T.delta_run(e).items():
            assert torch.equal(t, ref[k]), (how, k)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_parts_and_tokens(lib, dt):
    """A prompt, the same in two parts, and its last tokens one at a time."""
    from ttt_amd.delta import gated_delta, gated_delta_step
    d = T.delta_inputs(3, 90, 4, 2, 48, 64, dt, seed=4)
    q = {k: None if t is None else t.double() for k, t in d.items()}
    want, last = O.gated_delta(*(q[k] for k in ("q", "k", "v", "g", "beta", "state")))
    g = T.dev(d)
    tol = T.U * 40 * (1 + math.sqrt(90))

    def close(a, b, t, what):
        err = float((a.double().cpu() - b).norm() / b.norm())
        assert err <= tol + t, (what, err)

    out = T.half_step(dt) if dt != F32 else 0.0
    out += 2 * 2.0 ** -17 if dt == BF16 else 0.0
    for cut in (1, 17, 64, 89):
        args = lambda a, b: [g[k][:, a:b] for k in ("q", "k", "v", "g", "beta")]  # noqa: E731
        y1, s = gated_delta(*args(0, cut), g["state"], return_final_state=True)
        y2, s = gated_delta(*args(cut, 90), s, return_final_state=True)
        close(torch.cat([y1, y2], 1), want, out, cut)
        close(s, last, 0.0, cut)
    _, s = gated_delta(*args(0, 80), g["state"], return_final_state=True)
    ys = [gated_delta_step(*(g[k][:, t] for k in ("q", "k", "v", "g", "beta")), s) for t in range(80, 90)]
    close(torch.stack(ys, 1), want[:, 80:], out, "tokens")
    close(s, last, 0.0, "tokens")


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,H,G,N,P", [(1, 1, 1, 16, 32), (5, 6, 2, 80, 96), (64, 4, 4, 64, 64), (2, 3, 1, 128, 256)])
@pytest.mark.parametrize("unit", [True, False])
def test_step(lib, dt, B, H, G, N, P, unit):
    from ttt_amd.delta import gated_delta_step
    d = T.delta_inputs(B, 1, H, G, N, P, dt, seed=B + N, unit=unit)
    d["g"][0, 0, 0] = -math.inf
    q = {k: None if t is None else t.double() for k, t in d.items()}
    want, last = O.gated_delta(*(q[k] for k in ("q", "k", "v", "g", "beta", "state")), unit=unit)
    size = O.gated_delta_all(*(q[k] for k in ("q", "k", "v", "g", "beta", "state", "do", "dlast")), unit=unit, sizes=True)
    g = T.dev(d)
    s = g["state"].clone()
    y = gated_delta_step(*(g[k][:, 0] for k in ("q", "k", "v", "g", "beta")), s, l2_norm=unit)
    c = T.U * (8 + math.sqrt(N + P))
    T.within(y, want[:, 0], c * size["o"].norm() + (T.half_step(dt) * want.norm() if dt != F32 else 0), "o")
    T.within(s, last, c * size["last"].norm(), "state")


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_not_finite(lib, dt, which, bad):
    """A value that is not finite reaches its own sequence from its token on, no earlier output
    and no other sequence."""
    d = T.dev(T.delta_inputs(3, 150, 2, 1, 32, 64, dt, seed=8))
    ref = T.delta_run(d, grads=False)
    for t in (0, 37, 66, 149):
        e = dict(d)
        e[which] = d[which].clone()
        e[which][1, t].view(-1)[0] = bad
        got = T.delta_run(e, grads=False)
        for b in (0, 2):
            assert torch.equal(got["o"][b], ref["o"][b]) and torch.equal(got["last"][b], ref["last"][b])
        assert torch.equal(got["o"][1, :t], ref["o"][1, :t]), t
        o = got["o"][1].float()
        if which == "v":
            assert torch.isnan(o[t:, 0, 0]).all() and torch.equal(got["o"][1, :, :, 1:], ref["o"][1, :, :, 1:])
        elif which == "q":
            assert not torch.isfinite(o[t]).all() and torch.equal(got["o"][1, t + 1:], ref["o"][1, t + 1:])
        else:
            assert torch.isnan(o[t:, 0]).all() and torch.isnan(got["last"][1, 0]).all()


def test_largest_values(lib):
    """A value above what the products' planes hold, 3.39e38, counts as infinite whatever stands
    beside it: no earlier output sees it."""
    d = T.dev(T.delta_inputs(2, 100, 1, 1, 32, 32, F32, seed=13))
    d["beta"][:] = 1.0
    ref = T.delta_run(d, grads=False)
    for t in (5, 30, 70):
        for other in (-3.3e38, 3.3e38):
            e = {**d, "v": d["v"].clone()}
            e["v"][1, t, 0, 0], e["v"][1, t + 1, 0, 0] = 3.4e38, other
            got = T.delta_run(e, grads=False)
            assert torch.equal(got["o"][0], ref["o"][0]) and torch.equal(got["o"][1, :t], ref["o"][1, :t]), (t, other)
            assert torch.isnan(got["o"][1, t:, 0, 0]).all() and torch.equal(got["o"][1, :, :, 1:], ref["o"][1, :, :, 1:])


def test_empty(lib):
    from ttt_amd.delta import gated_delta, gated_delta_step
    for B, L in ((2, 0), (0, 5)):
        d = T.dev(T.delta_inputs(B, L, 2, 1, 32, 64, BF16))
        s = d["state"].requires_grad_(True)
        v = d["v"].detach().requires_grad_(True)
        o, last = gated_delta(d["q"], d["k"], v, d["g"], d["beta"], s, return_final_state=True)
        assert o.shape == (B, L, 2, 64) and torch.equal(last, s) and last is not s
        o.sum().backward()
        assert v.grad.shape == v.shape
        o, last = gated_delta(d["q"], d["k"], d["v"], d["g"], d["beta"], return_final_state=True)
        assert (last == 0).all()
    d = T.dev(T.delta_inputs(0, 1, 2, 1, 32, 64, BF16))
    assert gated_delta_step(*(d[k][:, 0] for k in ("q", "k", "v", "g", "beta")), d["state"]).shape == (0, 2, 64)


def test_partial_gradients(lib):
    """Gradients of some inputs alone, and of one output alone, are those of all."""
    from ttt_amd.delta import gated_delta
    d = T.dev(T.delta_inputs(2, 90, 4, 2, 32, 32, F32, seed=11))
    full = T.delta_run(d)
    v = d["v"].detach().requires_grad_(True)
    o, last = gated_delta(d["q"], d["k"], v, d["g"], d["beta"], d["state"], return_final_state=True)
    (g,) = torch.autograd.grad([o, last], v, [d["do"], d["dlast"]], retain_graph=True)
    assert torch.equal(g, full["dv"])
    (g1,) = torch.autograd.grad(o, v, d["do"], retain_graph=True)
    (g2,) = torch.autograd.grad(last, v, d["dlast"])
    torch.testing.assert_close(g1 + g2, full["dv"], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_expanded_and_repeated(lib, dt):
    """Inputs that a batch shares (stride 0) give the sum of their gradients, and a call gives the
    same bits every time."""
    d = T.dev(T.delta_inputs(3, 80, 4, 2, 32, 64, dt, seed=12))
    one = {k: d[k][:1].detach().clone().requires_grad_(True) for k in ("q", "k", "state")}
    e = {**d, **{k: t.expand(3, *t.shape[1:]) for k, t in one.items()}}
    from ttt_amd.delta import gated_delta
    o, last = gated_delta(e["q"], e["k"], e["v"], e["g"], e["beta"], e["state"], return_final_state=True)
    gs = torch.autograd.grad([o, last], list(one.values()), [d["do"], d["dlast"]])
    full = {**d, **{k: t.detach().expand(3, *t.shape[1:]).clone() for k, t in one.items()}}
    ref = T.delta_run(full)
    for k, g in zip(one, gs):
        torch.testing.assert_close(g.float(), ref["d" + k].float().sum(0, keepdim=True), rtol=2e-2 if dt != F32 else 1e-5,
                                   atol=2e-2 if dt != F32 else 1e-5)
    for k, t in T.delta_run(full).items():
        assert torch.equal(t, ref[k]), k


def test_on_another_stream_and_in_a_graph(lib):
    from ttt_amd.delta import gated_delta, gated_delta_step
    d = T.dev(T.delta_inputs(2, 300, 2, 1, 64, 64, BF16, seed=13))
    ref = T.delta_run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = T.delta_run(d)
    torch.cuda.current_stream().wait_stream(side)
    for k in ref:
        assert torch.equal(got[k], ref[k]), k
    args = [d[k].clone() for k in ("q", "k", "v", "g", "beta")]
    state = d["state"].clone()
    with torch.no_grad():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, last = gated_delta(*args, state, return_final_state=True)
            y = gated_delta_step(*(t[:, 0] for t in args), last)
        for seed in (14, 15, 16):
            e = T.dev(T.delta_inputs(2, 300, 2, 1, 64, 64, BF16, seed=seed))
            for a, k in zip(args, ("q", "k", "v", "g", "beta")):
                a.copy_(e[k])
            g.replay()
            wo, wl = gated_delta(*args, state, return_final_state=True)
            wy = gated_delta_step(*(t[:, 0] for t in args), wl)
            torch.cuda.synchronize()
            assert torch.equal(o, wo) and torch.equal(last, wl) and torch.equal(y, wy)


def test_saved_on_the_cpu(lib):
    d = T.dev(T.delta_inputs(2, 75, 4, 2, 64, 64, BF16, seed=17))
    ref = T.delta_run(d)
    with torch.autograd.graph.save_on_cpu():
        got = T.delta_run(d)
    for k in ref:
        assert torch.equal(got[k], ref[k]), k


def test_gradients_of_differences(lib):
    """The gradient along a direction against the difference of two calls, in fp32."""
    d = T.dev(T.delta_inputs(1, 70, 2, 1, 32, 32, F32, seed=18))
    got = T.delta_run(d)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for k in ("q", "k", "v", "g", "beta", "state"):
        dirn = torch.randn(d[k].shape, generator=gen, device="cuda") * d[k].abs().mean()
        h = 1e-2
        ys = []
        for s in (h, -h):
            e = T.delta_run({**d, k: d[k] + s * dirn}, grads=False)
            ys.append((e["o"].double() * d["do"]).sum() + (e["last"].double() * d["dlast"]).sum())
        want = float((got["d" + k].double() * dirn).sum())
        # a difference is off by its third derivative times h^2 and by fp32's rounding over h
        size = float((got["d" + k].double() * dirn).abs().sum())
        assert abs(float(ys[0] - ys[1]) / (2 * h) - want) <= 1e-3 * size + 1e-2 * abs(want), k
