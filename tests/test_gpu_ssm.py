"""The short causal convolution and the selective scan on the GPU against the plain
float64 forms, over sizes, types, layouts and states; a prompt in parts and token by
token; values that are not finite; graphs, streams and repeated calls."""

import math

import pytest
import torch

from tests import _ssm as T

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------
# convolution
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,L,C,W,act,state,pad", [
    (1, 1, 1, 2, None, False, 0), (2, 1, 8, 4, "silu", True, 0), (3, 2, 17, 4, "silu", False, 3),
    (2, 3, 64, 4, None, True, 8), (1, 15, 40, 3, "silu", True, 5), (2, 32, 129, 4, "silu", True, 1),
    (2, 33, 128, 2, "silu", False, 0), (1, 95, 7, 3, None, True, 0), (3, 200, 96, 4, "silu", True, 16),
    (1, 3001, 24, 4, "silu", True, 0), (70, 5, 33, 4, "silu", False, 0)])
def test_conv(lib, dt, B, L, C, W, act, state, pad):
    d = T.conv_inputs(B, L, C, W, dt, seed=B + L + C, state=state, pad=pad, bias=L != 95)
    T.conv_check(d, T.conv_run(T.dev(d), act), act)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_conv_in_parts_and_by_tokens(lib, dt):
    """A prompt, the same in two parts, and its last tokens one at a time: the same bits."""
    from ttt_amd.ssm import causal_conv, causal_conv_step
    d = T.dev(T.conv_inputs(3, 41, 50, 4, dt, seed=4))
    x, w, b, s0 = d["x"], d["weight"], d["bias"], d["state"]
    y, last = causal_conv(x, w, b, s0, "silu", True)
    for cut in (1, 2, 17, 40):
        y1, s = causal_conv(x[:, :cut], w, b, s0, "silu", True)
        y2, s = causal_conv(x[:, cut:], w, b, s, "silu", True)
        assert torch.equal(torch.cat([y1, y2], 1), y) and torch.equal(s, last)
    _, s = causal_conv(x[:, :30], w, b, s0, "silu", True)
    for t in range(30, 41):
        assert torch.equal(causal_conv_step(x[:, t], s, w, b, "silu"), y[:, t])
    assert torch.equal(s, last)


def test_conv_partial_gradients(lib):
    """Only the gradients that are asked for, and outputs of which one has none."""
    from ttt_amd.ssm import causal_conv
    d = T.dev(T.conv_inputs(2, 20, 16, 4, F32, seed=1))
    full = T.conv_run(d, "silu")
    x = d["x"].clone().requires_grad_(True)
    y, last = causal_conv(x, d["weight"], d["bias"], d["state"], "silu", True)
    (gy,) = torch.autograd.grad(y, x, d["dy"], retain_graph=True)
    (gl,) = torch.autograd.grad(last, x, d["dlast"])
    torch.testing.assert_close(gy + gl, full["dx"], rtol=1e-6, atol=1e-6)
    w = d["weight"].clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(causal_conv(d["x"], w, None, None, None), w, d["dy"])
    assert gw.shape == w.shape


# ---------------------------------------------------------------------------
# scan
# ---------------------------------------------------------------------------

SHAPES = [  # B, L, H, P, G, N
    (1, 1, 1, 32, 1, 16), (2, 2, 2, 64, 1, 64), (1, 31, 3, 32, 3, 48), (2, 32, 2, 64, 2, 32), (1, 33, 4, 64, 2, 128),
    (1, 63, 2, 32, 1, 64), (2, 64, 1, 64, 1, 80), (3, 65, 6, 64, 2, 64), (1, 129, 5, 32, 5, 16), (2, 200, 4, 64, 1, 96),
    (1, 333, 12, 64, 1, 64)]


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,L,H,P,G,N", SHAPES)
def test_scan(lib, dt, B, L, H, P, G, N):
    d = T.scan_inputs(B, L, H, P, G, N, dt, seed=B + L + N)
    T.scan_check(d, T.scan_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("state,skip,bias,softplus,dt32", [
    (False, False, False, True, False), (True, False, True, False, True), (False, True, False, True, True)])
def test_scan_options(lib, dt, state, skip, bias, softplus, dt32):
    d = T.scan_inputs(2, 70, 4, 64, 2, 64, dt, seed=5, state=state, skip=skip, bias=bias, dt_dtype=F32 if dt32 else None)
    if not softplus:
        d["dt"] = (0.05 * d["dt"].abs()).to(d["dt"].dtype)
        d["dt_bias"] = None if d["dt_bias"] is None else torch.full_like(d["dt_bias"], 0.01)
    T.scan_check(d, T.scan_run(T.dev(d), softplus), softplus)


@pytest.mark.parametrize("dt,L", [(BF16, 2500), (F32, 1300), (F16, 1500)])
def test_scan_long_single_sequence(lib, dt, L):
    """Few chains: the length is cut into segments."""
    d = T.scan_inputs(1, L, 2, 32, 1, 32, dt, seed=9)
    T.scan_check(d, T.scan_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_scan_many_chains(lib, dt):
    """As many chains as make one segment of each, heads in one pass of the backward."""
    d = T.scan_inputs(33, 140, 8, 32, 2, 16, dt, seed=10)
    T.scan_check(d, T.scan_run(T.dev(d)))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_scan_strong_and_weak_decays(lib, dt):
    """Tokens that forget everything among tokens that forget nothing: the factors behind
    a strong decay are as exact as any, and a step of 0 leaves the state as it is."""
    d = T.scan_inputs(1, 150, 4, 32, 1, 32, dt, seed=6, dt_dtype=F32, bias=False)
    d["dt"] = torch.full((1, 150, 4), -7.0)
    d["dt"][:, 10::23] = 40.0  # a decay of e^-600 and less
    d["dt"][:, 5::7] = -math.inf
    got = T.scan_run(T.dev(d))
    T.scan_check({**d, "dt": d["dt"].clamp(min=-1e4)}, got)
    assert (got["ddt"].cpu()[:, 5::7] == 0).all()
    only = {k: (t[:, :1] if k in ("x", "dt", "Bm", "Cm", "dy") else t) for k, t in d.items()}
    only["dt"] = torch.full((1, 1, 4), -math.inf)
    assert torch.equal(T.scan_run(T.dev(only), grads=False)["last"].cpu(), d["state"])


@pytest.mark.parametrize("dt", T.DTYPES)
def test_scan_layouts(lib, dt):
    """Columns of one matrix, contiguous tensors, rows that start off 16 bytes, expanded
    groups and transposed memory give the same bits."""
    d = T.dev(T.scan_inputs(2, 75, 4, 64, 2, 64, dt, seed=7))
    ref = T.scan_run(d)
    for how in ("contiguous", "odd rows", "transposed"):
        q = dict(d)
        for k in ("x", "Bm", "Cm", "dt"):
            t = d[k]
            if how == "contiguous":
                q[k] = t.contiguous()
            elif how == "odd rows":
                flat = t.flatten(2)
                m = torch.zeros(2, 75, flat.shape[2] + 3, device="cuda", dtype=t.dtype)
                m[..., 1:-2] = flat
                q[k] = m[..., 1:-2].unflatten(2, t.shape[2:])
            else:
                q[k] = t.transpose(0, 1).contiguous().transpose(0, 1)
        got = T.scan_run(q)
        for k in ref:
            assert torch.equal(got[k], ref[k]), (how, k)
    e = dict(d, Bm=d["Bm"][:, :, :1].expand(-1, -1, 2, -1))
    c = dict(e, Bm=e["Bm"].contiguous())
    for k, v in T.scan_run(e).items():
        assert torch.equal(v, T.scan_run(c)[k]), k


@pytest.mark.parametrize("dt", T.DTYPES)
def test_scan_sequences_do_not_mix(lib, dt):
    """The same sequence twice in a batch, beside others: the same bits."""
    d = T.scan_inputs(3, 90, 2, 64, 1, 64, dt, seed=8)
    for k in ("x", "dt", "Bm", "Cm", "state", "dy", "dlast"):
        d[k] = d[k].clone()
        d[k][2] = d[k][0]
    got = T.scan_run(T.dev(d))
    for k in ("y", "last", "dx", "ddt", "dBm", "dCm", "dstate"):
        assert torch.equal(got[k][0], got[k][2]), k


def test_scan_repeats(lib):
    """Two calls on the same inputs: the same bits (no atomic sums)."""
    d = T.dev(T.scan_inputs(2, 300, 6, 64, 1, 64, BF16, seed=11))
    a, b = T.scan_run(d), T.scan_run(d)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("P,N", [(64, 64), (32, 128)])
def test_scan_in_parts_and_by_tokens(lib, dt, P, N):
    """A prompt, the same in two parts, and its last tokens one at a time."""
    from ttt_amd.ssm import selective_scan, selective_scan_step
    c = T.scan_inputs(2, 150, 4, P, 2, N, dt, seed=12)
    d = T.dev(c)
    par = dict(D=d["D"], dt_bias=d["dt_bias"])
    ref, size = T.scan_reference(c, grads=False)

    def near(y, s, t0, t1, what):
        T.within(y, ref["y"][:, t0:t1], size["y"][:, t0:t1], 150 + P + N, what, None if dt == F32 else dt)
        if t1 == 150:
            T.within(s, ref["last"], size["last"], 150 + P + N, what)

    part = lambda t0, t1: [d[k][:, t0:t1] for k in ("x", "dt")] + [d["A"]] + [d[k][:, t0:t1] for k in ("Bm", "Cm")]  # noqa: E731
    for cut in (1, 64, 100, 149):
        y1, s = selective_scan(*part(0, cut), initial_state=d["state"], return_final_state=True, **par)
        y2, s = selective_scan(*part(cut, 150), initial_state=s, return_final_state=True, **par)
        near(torch.cat([y1, y2], 1), s, 0, 150, f"cut {cut}")
    _, s = selective_scan(*part(0, 130), initial_state=d["state"], return_final_state=True, **par)
    for t in range(130, 150):
        x, st, A, b, k = (v if v.dim() == 1 else v[:, 0] for v in part(t, t + 1))
        y = selective_scan_step(x, st, A, b, k, s, **par)
        near(y[:, None], s, t, t + 1, f"step {t}")


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,H,P,G,N", [(1, 1, 32, 1, 16), (5, 6, 64, 3, 48), (2, 4, 32, 1, 112), (64, 12, 64, 1, 64)])
def test_scan_step(lib, dt, B, H, P, G, N):
    from ttt_amd.ssm import selective_scan_step
    c = T.scan_inputs(B, 1, H, P, G, N, dt, seed=B + N)
    ref, size = T.scan_reference(c, grads=False)
    d = T.dev(c)
    s = d["state"].clone()
    y = selective_scan_step(d["x"][:, 0], d["dt"][:, 0], d["A"], d["Bm"][:, 0], d["Cm"][:, 0], s, D=d["D"],
                            dt_bias=d["dt_bias"])
    T.within(y, ref["y"][:, 0], size["y"][:, 0], N, "y", None if dt == F32 else dt)
    T.within(s, ref["last"], size["last"], 1, "state")


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("t", [0, 5, 16, 47, 63, 64, 100])
def test_scan_not_finite_from_its_token_on(lib, dt, bad, t):
    """One value that is not finite: the outputs before its token, of other features and
    of other sequences are as without it; its own from there on are not finite."""
    d = T.scan_inputs(2, 130, 2, 64, 1, 64, dt, seed=13)
    ref = T.scan_run(T.dev(d), grads=False)
    d["x"] = d["x"].clone()
    d["x"][1, t, 1, 37] = bad
    got = T.scan_run(T.dev(d), grads=False)
    hit = torch.zeros_like(ref["y"], dtype=torch.bool)
    hit[1, t:, 1, 37] = True
    assert torch.equal(got["y"][~hit], ref["y"][~hit])
    assert not torch.isfinite(got["y"][hit]).any()
    for k in ("Bm", "Cm", "dt"):
        q = {n: None if v is None else v.clone() for n, v in d.items()}
        q["x"][1, t, 1, 37] = 1.0
        q[k][1, t, 0] = bad
        base = dict(q)
        base[k] = d[k].clone()
        r = T.scan_run(T.dev(base), grads=False)["y"]
        y = T.scan_run(T.dev(q), grads=False)["y"]
        assert torch.equal(y[0], r[0]) and torch.equal(y[1, :t], r[1, :t]), k


def test_scan_gradient_of_a_direction(lib):
    """The fp32 gradients against differences of the float64 form along a direction: the
    two agree to the difference's own error, h^2 of the third derivative, and the kernels'."""
    from oracle import ssm_oracle as S
    d = T.scan_inputs(2, 70, 4, 32, 2, 32, F32, seed=14)
    got = T.scan_run(T.dev(d))
    g = torch.Generator().manual_seed(15)
    q = {k: d[k].double() for k in T.SCAN_ARGS}
    for k in T.SCAN_ARGS:
        v = torch.randn(q[k].shape, generator=g, dtype=torch.float64)
        h = 1e-6

        def loss(s):
            y, last = S.selective_scan(*[q[n] + (s * v if n == k else 0) for n in T.SCAN_ARGS])
            return (y * d["dy"].double()).sum() + (last * d["dlast"].double()).sum()

        want = float((loss(h) - loss(-h)) / (2 * h))
        have = float((got["d" + k].double().cpu() * v).sum())
        scale = float(got["d" + k].double().norm() * v.norm())
        assert abs(have - want) <= 1e-5 * scale, (k, have, want)


# ---------------------------------------------------------------------------
# graphs, streams, memory
# ---------------------------------------------------------------------------

def _train(d):
    return T.scan_run(d) | {"c" + k: v for k, v in T.conv_run({
        "x": d["x"].flatten(2), "weight": d["w"], "bias": None, "state": None, "dy": d["dy"].flatten(2),
        "dlast": d["dl"]}, "silu").items()}


def test_graph_replays(lib):
    """Forward and backward in one graph, replayed on new inputs between eager calls."""
    d = T.dev(T.scan_inputs(2, 190, 4, 64, 1, 64, BF16, seed=20))
    d["w"], d["dl"] = torch.randn(256, 4, device="cuda"), torch.randn(2, 3, 256, device="cuda").to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _train(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _train(d)
    for seed in (21, 22, 23, 24):
        new = T.dev(T.scan_inputs(2, 190, 4, 64, 1, 64, BF16, seed=seed))
        with torch.no_grad():
            for k, t in new.items():
                d[k].copy_(t)
        want = _train({**new, "w": d["w"], "dl": d["dl"]})
        torch.cuda.synchronize()
        graph.replay()
        got = {k: v.clone() for k, v in out.items()}
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), (seed, k)


def test_graph_of_a_token(lib):
    """A token's step in a graph: replays move the states on as eager calls do."""
    from ttt_amd.ssm import causal_conv_step, selective_scan_step
    d = T.dev(T.scan_inputs(3, 8, 4, 64, 1, 64, BF16, seed=25))
    w = torch.randn(256, 4, device="cuda")

    def token(t, cs, hs):
        x = causal_conv_step(t["x"].flatten(1), cs, w, None, "silu").view(3, 4, 64)
        return selective_scan_step(x, t["dt"], d["A"], t["Bm"], t["Cm"], hs, D=d["D"], dt_bias=d["dt_bias"])

    at = lambda i: {k: d[k][:, i].contiguous() for k in ("x", "dt", "Bm", "Cm")}  # noqa: E731
    buf = at(0)
    cs, hs = torch.zeros(3, 3, 256, device="cuda", dtype=BF16), d["state"].clone()
    graph = torch.cuda.CUDAGraph()
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        token(buf, cs.clone(), hs.clone())
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = token(buf, cs, hs)
    ecs, ehs = torch.zeros_like(cs), d["state"].clone()
    for i in range(8):
        for k, t in at(i).items():
            buf[k].copy_(t)
        graph.replay()
        want = token(at(i), ecs, ehs)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(cs, ecs) and torch.equal(hs, ehs), i


def test_two_streams(lib):
    """Two calls at once on two streams: each has its own workspace."""
    ds = [T.dev(T.scan_inputs(1, 900, 3, 64, 1, 64, BF16, seed=s)) for s in (30, 31)]
    want = [T.scan_run(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    for _ in range(3):
        got = []
        for d, s in zip(ds, streams):
            with torch.cuda.stream(s):
                got.append(T.scan_run(d))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            for k in w:
                assert torch.equal(w[k], g[k]), k


def test_writes_stay_inside(lib):
    """States behind the last sequence of a step are left as they were."""
    from ttt_amd.ssm import causal_conv_step, selective_scan_step
    d = T.dev(T.scan_inputs(3, 1, 3, 32, 1, 48, BF16, seed=33))
    pool = torch.full((5, 3, 32, 48), 7.0, device="cuda")
    s = pool[1:4]
    s.zero_()
    selective_scan_step(d["x"][:, 0], d["dt"][:, 0], d["A"], d["Bm"][:, 0], d["Cm"][:, 0], s)
    assert (pool[0] == 7).all() and (pool[4] == 7).all() and (s != 0).any()
    cpool = torch.full((5, 3, 33), 7.0, device="cuda", dtype=BF16)
    causal_conv_step(torch.ones(3, 33, device="cuda", dtype=BF16), cpool[1:4], torch.ones(33, 4, device="cuda"))
    assert (cpool[0] == 7).all() and (cpool[4] == 7).all() and (cpool[1:4, 2] == 1).all()


def test_empty(lib):
    from ttt_amd.ssm import causal_conv, selective_scan
    d = T.dev(T.scan_inputs(2, 3, 2, 32, 1, 16, BF16, seed=1))
    y, s = selective_scan(d["x"][:, :0], d["dt"][:, :0], d["A"], d["Bm"][:, :0], d["Cm"][:, :0],
                          initial_state=d["state"], return_final_state=True)
    assert y.shape == (2, 0, 2, 32) and torch.equal(s, d["state"])
    y, s = causal_conv(torch.empty(2, 0, 5, device="cuda"), torch.ones(5, 3, device="cuda"), return_final_state=True)
    assert y.shape == (2, 0, 5) and s.shape == (2, 2, 5) and (s == 0).all()


def test_empty_gradients(lib):
    """No tokens: no gradient of the parameters, and the state's passes through."""
    from ttt_amd.norm import layer_norm
    from ttt_amd.ssm import causal_conv, selective_scan
    d = T.dev(T.scan_inputs(2, 3, 2, 32, 1, 16, BF16, seed=1))
    a, s0 = (d[k].clone().requires_grad_(True) for k in ("A", "state"))
    y, s = selective_scan(d["x"][:, :0], d["dt"][:, :0], a, d["Bm"][:, :0], d["Cm"][:, :0], initial_state=s0,
                          return_final_state=True)
    ga, gs = torch.autograd.grad(y.sum() + 2 * s.sum(), [a, s0])
    assert (ga == 0).all() and (gs == 2).all()
    w = torch.ones(5, 3, device="cuda", requires_grad=True)
    y = causal_conv(torch.empty(2, 0, 5, device="cuda"), w)
    assert (torch.autograd.grad(y.sum(), w)[0] == 0).all()
    w, b = (torch.ones(5, device="cuda", requires_grad=True) for _ in range(2))
    y = layer_norm(torch.empty(0, 5, device="cuda"), w, b)
    assert all((g == 0).all() for g in torch.autograd.grad(y.sum(), [w, b]))
    with pytest.raises(ValueError, match="weight"):
        causal_conv(torch.empty(2, 0, 5, device="cuda"), torch.ones(4, 3, device="cuda"))
    with pytest.raises(ValueError, match="initial_state"):
        selective_scan(d["x"][:, :0], d["dt"][:, :0], d["A"], d["Bm"][:, :0], d["Cm"][:, :0],
                       initial_state=d["state"][:1])


@pytest.mark.parametrize("L", [1, 2])
def test_scan_of_rows_far_apart(lib, L):
    """Rows 64 MiB apart: of different sequences where they are tokens alone, and of one."""
    from ttt_amd.ssm import selective_scan
    B = 3 - L
    d = T.dev(T.scan_inputs(B, L, 2, 32, 1, 16, BF16, seed=2))
    wide = torch.empty(B * L, (1 << 25) + 8, device="cuda", dtype=BF16)
    x = wide[:, :64].view(B, L, 2, 32)
    x.copy_(d["x"])
    a = [d[k].clone().requires_grad_(True) if k == "A" else d[k] for k in ("dt", "A", "Bm", "Cm")]
    g = wide[:, 64:128].view(B, L, 2, 32)
    g.copy_(d["x"])
    want, y = selective_scan(d["x"].contiguous(), *a), selective_scan(x, *a)
    assert torch.equal(y, want)
    assert torch.equal(*(torch.autograd.grad(o, a[1], t)[0] for o, t in ((y, g), (want, d["x"].contiguous()))))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_conv_of_a_large_batch(lib, dt):
    """A thread's run is longer in a large batch: a sequence's values are the same bits alone."""
    from ttt_amd.ssm import causal_conv
    torch.manual_seed(3)
    x, w = torch.randn(33, 1031, 521, device="cuda").to(dt), torch.randn(521, 4, device="cuda")
    y, last = causal_conv(x, w, None, None, "silu", True)
    for b in (0, 17, 32):
        y1, last1 = causal_conv(x[b:b + 1], w, None, None, "silu", True)
        assert torch.equal(y[b:b + 1], y1) and torch.equal(last[b:b + 1], last1)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_skip_gradient_over_many_tokens(lib, dt):
    """dD is a sum of 131,072 products a head.  In steps rounded to nearest its error is that of
    sums of 1,024 of them, 15 roundings of half a step of 2^-24 each: relative to the root of
    the sum of the squares, the root of 15 half steps, and no more for more tokens; twice the
    root is 8."""
    from ttt_amd.ssm import selective_scan
    torch.manual_seed(5)
    B, L, H, P, N = 8, 512, 8, 32, 32
    x, dy = (torch.randn(B, L, H, P, device="cuda").to(dt) for _ in range(2))
    b, c = (torch.randn(B, L, 1, N, device="cuda").to(dt) for _ in range(2))
    D = torch.ones(H, device="cuda", requires_grad=True)
    y = selective_scan(x, torch.zeros(B, L, H, device="cuda").to(dt), -torch.ones(H, device="cuda"), b, c, D)
    (got,) = torch.autograd.grad(y, D, dy)
    terms = (x.double() * dy.double()).permute(2, 0, 1, 3).flatten(1)
    assert ((got.double() - terms.sum(1)).abs() <= 8 * 2.0 ** -24 * terms.square().sum(1).sqrt()).all()


def test_offsets_past_32_bits(lib):
    """Rows of a matrix of more than 4 GiB: the same bits as from rows of their own."""
    from ttt_amd.norm import layer_norm
    from ttt_amd.ssm import causal_conv, selective_scan
    B, L, ld = 2, 70000, 16400
    wide = torch.empty(B, L, ld, device="cuda", dtype=BF16)
    assert wide.numel() * 2 > 1 << 32
    xbc = wide[..., 8:8 + 96]
    xbc.copy_(torch.randn(B, L, 96, device="cuda"))
    own = xbc.contiguous()
    w = torch.randn(96, 4, device="cuda")
    conv = [causal_conv(t, w, None, None, "silu", True) for t in (xbc, own)]
    assert all(torch.equal(a, b) for a, b in zip(*conv))
    norm = [layer_norm(t, gate=t) for t in (xbc, own)]
    assert torch.equal(*norm)
    A = -torch.ones(2, device="cuda")

    def scan(t):
        x = t.detach().requires_grad_(True)
        y = selective_scan(x[..., :64].unflatten(-1, (2, 32)), x[..., 64:66], A, x[..., 64:80].unflatten(-1, (1, 16)),
                           x[..., 80:].unflatten(-1, (1, 16)))
        return y, torch.autograd.grad(y, x, y.detach())[0]

    for a, b in zip(scan(xbc), scan(own)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("P,N,dt", [(64, 128, F32), (32, 128, F16), (64, 128, BF16)])
def test_graph_of_large_workgroups(lib, P, N, dt):
    """Kernels of more than 64 KB of LDS and of many segments, in a graph."""
    d = T.dev(T.scan_inputs(1, 1500, 2, P, 1, N, dt, seed=40))
    want = T.scan_run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        T.scan_run(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = T.scan_run(d)
    for _ in range(3):
        for v in got.values():
            v.zero_()
        graph.replay()
        again = T.scan_run(d)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]) and torch.equal(again[k], want[k]), k


def test_inference_mode(lib):
    from ttt_amd.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    d = T.dev(T.scan_inputs(2, 9, 2, 32, 1, 16, BF16, seed=41))
    w = torch.randn(64, 4, device="cuda")

    def run():
        x, s = causal_conv(d["x"].flatten(2), w, None, None, "silu", True)
        _, h = selective_scan(x.unflatten(-1, (2, 32)), d["dt"], d["A"], d["Bm"], d["Cm"], return_final_state=True)
        x = causal_conv_step(d["x"][:, 0].flatten(1), s, w, None, "silu")
        y = selective_scan_step(x.unflatten(-1, (2, 32)), d["dt"][:, 0], d["A"], d["Bm"][:, 0], d["Cm"][:, 0], h)
        return y, s, h

    with torch.no_grad():
        want = run()
    with torch.inference_mode():
        got = run()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
