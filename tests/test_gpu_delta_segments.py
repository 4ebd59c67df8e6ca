"""The gated delta rule where a sequence is cut into segments, as long prompts of few heads are: values
that are not finite, weights and decays at their ends, prompts in parts, layouts, streams, graphs and
hooks on saved tensors.  Each test sees in the workspace's size that there are segments."""

import math

import pytest
import torch

from oracle import block_oracle as O
from tests import _block as T

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CHUNK, TILES, CODE = {BF16: 64, F16: 32, F32: 32}, {BF16: 10, F16: 3, F32: 3}, {F32: 0, BF16: 1, F16: 2}


def segments(lib, d):
    """How many segments the library cuts these inputs into, from the bytes beside Z, M and the tokens' numbers"""
    (B, L, H, P), N, dt = d["v"].shape, d["k"].shape[-1], d["v"].dtype
    Q = CHUNK[dt]
    NC, NP = -(-L // Q), 32 if N <= 32 else 64 if N <= 64 else 128
    tok = -(-B * H * NC * (8 * Q + 4) * 4 // 256) * 256
    S, odd = divmod(lib.ttt_delta_workspace_bytes(B, L, H, P, N, CODE[dt]) - tok - 2 * B * H * NC * TILES[dt] * 1024,
                    B * H * 4 * NP * (P + NP))
    assert odd == 0 and S > 2, S
    return S, -(-NC // S) * Q


def inputs(lib, *a, **kw):
    d = T.delta_inputs(*a, **kw)
    segments(lib, d)
    return d


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("N,P", [(32, 64), (128, 32)])
def test_not_finite(lib, dt, which, bad, N, P):
    """A value that is not finite, in the first, a middle and the last segment and on both sides of their
    borders, reaches its own sequence from its token on, no earlier output and no other sequence."""
    d = T.dev(T.delta_inputs(2, 900, 2, 1, N, P, dt, seed=8))
    S, per = segments(lib, d)
    ref = T.delta_run(d, grads=False)
    for t in (0,) if which == "state" else (0, 5, per - 1, per, (S // 2) * per + 7, 899):
        e = dict(d)
        e[which] = d[which].clone()
        (e[which][1] if which == "state" else e[which][1, t]).view(-1)[0] = bad
        got = T.delta_run(e, grads=False)
        assert torch.equal(got["o"][0], ref["o"][0]) and torch.equal(got["last"][0], ref["last"][0]), t
        assert torch.equal(got["o"][1, :t], ref["o"][1, :t]), t
        o, want = got["o"][1], ref["o"][1]
        if which in ("v", "state"):  # its own feature alone
            assert torch.isnan(o[max(t, 1):, 0, 0]).all() and not torch.isfinite(o[t, 0, 0]), t
            assert torch.equal(o[:, 1], want[:, 1]) and torch.equal(o[:, 0, 1:], want[:, 0, 1:]), t
            assert torch.isnan(got["last"][1, 0, 0]).all() and torch.equal(got["last"][1, 0, 1:], ref["last"][1, 0, 1:]), t
        elif which == "q":
            assert not torch.isfinite(o[t]).all() and torch.equal(o[t + 1:], want[t + 1:]), t
            assert torch.equal(got["last"], ref["last"]), t
        else:
            assert torch.isnan(o[t:, 0]).all() and torch.isnan(got["last"][1, 0]).all(), t


def test_largest_values(lib):
    """An fp32 value above 3.39e38 counts as infinite: no earlier output sees it."""
    d = T.dev(T.delta_inputs(2, 700, 1, 1, 32, 32, F32, seed=13))
    S, per = segments(lib, d)
    d["beta"][:] = 1.0
    ref = T.delta_run(d, grads=False)
    for t in (5, per - 1, per, (S - 1) * per + 3):
        for other in (-3.3e38, 3.3e38):
            e = {**d, "v": d["v"].clone()}
            e["v"][1, t, 0, 0], e["v"][1, t + 1, 0, 0] = 3.4e38, other
            got = T.delta_run(e, grads=False)
            assert torch.equal(got["o"][0], ref["o"][0]) and torch.equal(got["o"][1, :t], ref["o"][1, :t]), (t, other)
            assert torch.isnan(got["o"][1, t:, 0, 0]).all() and torch.equal(got["o"][1, :, :, 1:], ref["o"][1, :, :, 1:])


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("N,P", [(32, 64), (64, 64), (128, 128)])
def test_weights_and_decays_at_their_ends(lib, dt, N, P):
    """Weights of 0 and 1, decays of 0, of e^-600 and of nothing left, at the borders of segments too;
    keys that repeat."""
    d = T.delta_inputs(1, 900, 2, 2, N, P, dt, seed=6)
    _, per = segments(lib, d)
    d["beta"][:, 3::7] = 0.0
    d["beta"][:, 5::11] = 1.0
    d["g"][:, ::5] = 0.0
    d["g"][:, 110::230] = -600.0
    d["g"][:, per], d["g"][:, 2 * per - 1], d["g"][:, 417] = -math.inf, -math.inf, -math.inf
    d["k"] = d["k"].clone()
    d["k"][:, 40:60] = d["k"][:, 40:41]
    got = T.delta_run(T.dev(d))
    T.delta_check({**d, "g": d["g"].clamp(min=-1e4)}, got)
    assert (got["dv"].cpu()[d["beta"] == 0] == 0).all()


@pytest.mark.parametrize("dt", T.DTYPES)
def test_a_state_that_is_forgotten(lib, dt):
    """With g = -inf at the first token of a segment, and inside one, nothing of what was before it is left, a
    value of fp32's largest in the state included: the last state is that of a call that begins there."""
    d = T.dev(T.delta_inputs(1, 900, 2, 1, 32, 64, dt, seed=7))
    _, per = segments(lib, d)
    for t in (per, per + 21):
        e = {**d, "g": d["g"].clone(), "state": d["state"] * 1e30}
        e["g"][:, t] = -math.inf
        got = T.delta_run(e, grads=False)
        tail = {k: d[k][:, t:].cpu() for k in ("q", "k", "v", "beta", "do")}
        tail.update(g=e["g"][:, t:].clamp(min=-1e4).cpu(), state=torch.zeros_like(d["state"]).cpu(), dlast=d["dlast"].cpu())
        T.delta_check(tail, {"o": got["o"][:, t:], "last": got["last"]})


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("state,unit,scale", [(False, False, None), (True, False, 0.7), (False, True, 1.0)])
def test_options(lib, dt, state, unit, scale):
    d = inputs(lib, 1, 900, 2, 1, 48, 96, dt, seed=5, state=state, unit=unit, g_dtype=dt, beta_dtype=dt)
    T.delta_check(d, T.delta_run(T.dev(d), unit, scale), unit, scale)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_layouts(lib, dt):
    """Columns of one matrix, contiguous tensors, rows off 16 bytes and transposed memory give the same bits."""
    d = T.dev(inputs(lib, 2, 875, 2, 2, 64, 64, dt, seed=7))
    ref = T.delta_run(d)
    for how in ("contiguous", "odd rows", "transposed"):
        e = dict(d)
        for k in ("q", "k", "v", "g", "beta"):
            t = d[k]
            if how == "contiguous":
                e[k] = t.contiguous()
            elif how == "odd rows":
                flat = t.flatten(2)
                m = torch.zeros(2, 875, flat.shape[2] + 3, device="cuda", dtype=t.dtype)
                m[..., 1:-2] = flat
                e[k] = m[..., 1:-2].unflatten(2, t.shape[2:])
            else:
                e[k] = t.transpose(0, 1).contiguous().transpose(0, 1)
        e["do"] = d["do"].transpose(0, 1).contiguous().transpose(0, 1) if how == "transposed" else d["do"]
        for k, t in T.delta_run(e).items():
            assert torch.equal(t, ref[k]), (how, k)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_parts_and_tokens(lib, dt):
    """A prompt in two parts, cut inside a segment and at its border, and its last tokens one at a time."""
    from ttt_amd.delta import gated_delta, gated_delta_step
    d = T.delta_inputs(1, 900, 2, 1, 48, 64, dt, seed=4)
    _, per = segments(lib, d)
    q = {k: t.double() for k, t in d.items()}
    want, last = O.gated_delta(*(q[k] for k in T.DELTA_ARGS))
    g = T.dev(d)
    tol = T.U * 40 * (1 + math.sqrt(900))  # (half a step a factor, errors of L tokens like the root of L, as in the bound of one call)
    out = tol + (T.half_step(dt) if dt != F32 else 0.0) + (2 * 2.0 ** -17 if dt == BF16 else 0.0)

    def close(a, b, t, what):
        err = float((a.double().cpu() - b).norm() / b.norm())
        assert err <= t, (what, err)

    args = lambda a, b: [g[k][:, a:b] for k in ("q", "k", "v", "g", "beta")]  # noqa: E731
    for cut in (1, per, per + 17, 899):
        y1, s = gated_delta(*args(0, cut), g["state"], return_final_state=True)
        y2, s = gated_delta(*args(cut, 900), s, return_final_state=True)
        close(torch.cat([y1, y2], 1), want, out, cut)
        close(s, last, tol, cut)
    _, s = gated_delta(*args(0, 890), g["state"], return_final_state=True)
    ys = [gated_delta_step(*(g[k][:, t] for k in ("q", "k", "v", "g", "beta")), s) for t in range(890, 900)]
    close(torch.stack(ys, 1), want[:, 890:], out, "tokens")
    close(s, last, tol, "tokens")


@pytest.mark.parametrize("dt", T.DTYPES)
def test_again_on_another_stream_and_on_the_cpu(lib, dt):
    """The same bits in a second call, on another stream and with what was saved brought back from the CPU."""
    d = T.dev(inputs(lib, 1, 900, 2, 1, 64, 64, dt, seed=13))
    ref = T.delta_run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = T.delta_run(d)
    torch.cuda.current_stream().wait_stream(side)
    with torch.autograd.graph.save_on_cpu():
        back = T.delta_run(d)
    for got in (T.delta_run(d), other, back):
        for k in ref:
            assert torch.equal(got[k], ref[k]), k


@pytest.mark.parametrize("dt", T.DTYPES)
def test_in_a_graph(lib, dt):
    """Forward and backward captured once and replayed, other calls between the replays."""
    from ttt_amd.delta import gated_delta
    shape = (1, 900, 2, 1, 64, 64, dt)
    d = T.dev(inputs(lib, *shape, seed=14))
    leaves = [d[k].detach().clone().requires_grad_(True) for k in T.DELTA_ARGS]
    do, dlast = d["do"].clone(), d["dlast"].clone()

    def call():
        outs = gated_delta(*leaves, return_final_state=True)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [do, dlast]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (15, 16, 17):
        e = T.dev(T.delta_inputs(*shape, seed=seed))
        with torch.no_grad():
            for t, k in zip(leaves + [do, dlast], (*T.DELTA_ARGS, "do", "dlast")):
                t.copy_(e[k])
        graph.replay()
        want = T.delta_run(e)
        torch.cuda.synchronize()
        for t, (k, w) in zip(got, want.items()):
            assert torch.equal(t, w), (seed, k)
