"""What a gated delta-rule block's operators refuse, without a GPU: the C entry points return
their status before any launch, the Python ones raise."""

import pytest
import torch

from tests.test_ssm_refusals import BF16, E_ALIGN, E_ARG, E_DTYPE, E_NULL, E_SHAPE, E_WS, F16, F32, P, Q, _call

DELTA_IN = dict(q=P, ldq=128, k=P, ldk=128, v=P, ldv=256, g=P, ldg=4, beta=P, ldb=4)
DIMS = dict(B=2, L=99, H=4, P=64, G=2, N=64)
HOW = dict(scale=0.125, unit=1, dtype=BF16, gd=F32, bd=BF16)
DELTA = dict(**DELTA_IN, h0=P, **DIMS, **HOW, o=P, last=P, saved=P, sbytes=1 << 40, ws=P, wbytes=1 << 40, stream=None)
DELTA_BWD = dict(q=P, ldq=128, k=P, ldk=128, g=P, ldg=4, beta=P, ldb=4, dO=P, lddo=256, dlast=P, saved=P, sbytes=1 << 40,
                 kept=P, kbytes=1 << 40, **DIMS, **HOW, dq=P, dk=P, dv=P, dg=P, db=P, dh0=P, ws=P, wbytes=1 << 40, stream=None)
DELTA_STEP = dict(**DELTA_IN, h=P, B=2, H=4, P=64, G=2, N=64, **HOW, o=P, stream=None)
NORM = dict(x=P, ldx=64, gate=P, ldg=64, res=P, ldr=64, w=P, s=P, w2=P, R=6, D=64, heads=1, eps=1e-6, dtype=BF16, rd=F32,
            r=P, y=P, stats=P, stream=None)
NORM_BWD = dict(x=P, ldx=64, gate=P, ldg=64, res=P, ldr=64, w=P, s=P, w2=P, stats=P, dr=P, dy=P, R=6, D=64, heads=1,
                dtype=BF16, rd=F32, dx=P, dg=P, dres=P, dw=P, ds=P, dw2=P, part=P, bytes=1 << 30, stream=None)
FFN = dict(x=P, ldx=64, wg=P, wu=P, bg=P, bu=P, R=100, D=64, F=48, act=1, dtype=BF16, y=P, ws=P, bytes=1 << 40, stream=None)
FFN_BWD = dict(x=P, ldx=64, wg=P, wu=P, bg=P, bu=P, dy=P, lddy=48, R=100, D=64, F=48, act=1, dtype=BF16, dx=P, dwg=P, dwu=P,
               dbg=P, dbu=P, ws=P, bytes=1 << 40, stream=None)


@pytest.fixture(scope="module")
def lib():
    from ttt_amd import _lib
    return _lib.load()


def test_delta(lib):
    f, b, s = (lambda **kw: _call(lib.ttt_delta_fwd, DELTA, **kw)), (lambda **kw: _call(lib.ttt_delta_bwd, DELTA_BWD, **kw)), \
        (lambda **kw: _call(lib.ttt_delta_step, DELTA_STEP, **kw))
    for c in (f, b, s):
        for bad in (dict(P=48), dict(P=0), dict(P=288), dict(N=8), dict(N=72), dict(N=144), dict(G=3), dict(G=0), dict(H=0),
                    dict(B=0), dict(B=-1), dict(ldq=120), dict(ldk=120), dict(ldg=3), dict(ldb=3)):
            assert c(**bad) == E_SHAPE, bad
        assert c(dtype=3) == E_DTYPE and c(gd=F16) == E_DTYPE and c(bd=F16) == E_DTYPE
        for p in ("q", "k", "g", "beta"):
            assert c(**{p: None}) == E_NULL and c(**{p: P + 1}) == E_ALIGN, p
    assert f(ldv=255) == E_SHAPE and s(ldv=255) == E_SHAPE and b(lddo=255) == E_SHAPE
    for c in (f, b):
        assert c(L=0) == E_SHAPE and c(L=0x7fffffff) == E_SHAPE and c(ldq=132) == E_SHAPE and c(q=Q) == E_ALIGN
        assert c(ldk=1 << 25) == E_SHAPE and c(ldk=1 << 25, L=1, q=None) == E_NULL  # rows of a chunk out of reach
        assert c(B=1 << 20, L=1 << 16) == E_SHAPE and c(H=1 << 18) == E_SHAPE
        assert c(ws=None) == E_WS and c(ws=Q) == E_ALIGN and c(saved=Q) == E_ALIGN
    assert b(saved=None) == E_NULL and s(h=None) == E_NULL and s(h=Q) == E_ALIGN and s(ldq=130) == E_SHAPE and s(B=1 << 24) == E_SHAPE
    dims = (2, 99, 4, 64, 64, BF16)
    assert f(wbytes=lib.ttt_delta_workspace_bytes(*dims) - 1) == E_WS
    assert f(sbytes=lib.ttt_delta_saved_bytes(*dims) - 1) == E_WS and b(sbytes=lib.ttt_delta_saved_bytes(*dims) - 1) == E_WS
    assert b(kept=None) == E_NULL and b(kept=Q) == E_ALIGN and b(kbytes=4 * 2 * 4 * 2 * (516 + 2 * 2560) - 1) == E_WS
    assert b(wbytes=lib.ttt_delta_bwd_workspace_bytes(2, 99, 4, 64, 2, 64, BF16) - 1) == E_WS
    assert lib.ttt_delta_saved_bytes(2, 99, 4, 48, 64, BF16) == 0 and lib.ttt_delta_workspace_bytes(2, 99, 4, 64, 8, BF16) == 0
    assert lib.ttt_delta_bwd_workspace_bytes(2, 99, 4, 64, 3, 64, BF16) == 0


def test_delta_most_sequences(lib):
    """A launch has at most 2^32 - 1 threads, 8 to a feature and column of a state (128 at most), or
    up to 32 to a feature alone: refused past that."""
    for fn, more in ((lib.ttt_delta_saved_bytes, ()), (lib.ttt_delta_workspace_bytes, ()), (lib.ttt_delta_bwd_workspace_bytes, (1,))):
        for P, most in ((32, ((1 << 29) - 1) // 160), (64, (1 << 21) - 1), (256, (1 << 19) - 1)):
            assert fn(most, 1, 1, P, *more, 16, BF16) > 0
            assert fn(most + 1, 1, 1, P, *more, 16, BF16) == 0


def test_delta_segments_and_sizes(lib):
    """Sizes grow with what they are of, and a long prompt of few heads is cut into segments while
    many are not: the workspace beside Z, M and the tokens' numbers is the segments'."""
    for dt, Q, tiles in ((BF16, 64, 10), (F16, 32, 3), (F32, 32, 3)):
        for B, L, H, Pd, N in ((1, 16384, 12, 64, 64), (64, 2048, 12, 64, 64), (1, 1, 1, 32, 16), (3, 777, 4, 32, 32)):
            NC, NP = -(-L // Q), 32 if N <= 32 else 64
            tok = -(-B * H * NC * (8 * Q + 4) * 4 // 256) * 256
            rest = lib.ttt_delta_workspace_bytes(B, L, H, Pd, N, dt) - tok - 2 * B * H * NC * tiles * 1024
            S, odd = divmod(rest, B * H * 4 * NP * (Pd + NP))
            assert odd == 0 and (S == 0 or 2 <= S <= NC), (B, L, H, dt, S)
            assert (S > 4) == (B * H <= 12 and L > 700), (B, L, H, dt, S)
            assert lib.ttt_delta_saved_bytes(B, L, H, Pd, N, dt) == B * H * NC * Pd * 4 * (NP + Q)


def test_block_norm(lib):
    f, b = (lambda **kw: _call(lib.ttt_block_norm_fwd, NORM, **kw)), (lambda **kw: _call(lib.ttt_block_norm_bwd, NORM_BWD, **kw))
    for c in (f, b):
        for bad in (dict(R=0), dict(R=1 << 32), dict(D=0), dict(D=8193, ldx=1 << 14, ldg=1 << 14, ldr=1 << 14), dict(heads=0),
                    dict(heads=4), dict(heads=2), dict(ldx=63), dict(ldg=63), dict(ldr=63)):
            assert c(**bad) == E_SHAPE, bad
        assert c(dtype=3) == E_DTYPE and c(rd=F16) == E_DTYPE and c(dtype=F32, rd=BF16) == E_DTYPE
        assert c(rd=-1) == E_ARG  # a next norm without a residual
        assert c(x=None) == E_NULL and c(res=None) == E_NULL and c(x=P + 1) == E_ALIGN and c(w=P + 2) == E_ALIGN
    assert f(eps=0.0) == E_ARG and f(eps=2.0) == E_ARG and f(eps=float("nan")) == E_ARG
    assert f(w2=None, rd=-1) == E_ARG and f(r=None) == E_NULL and f(y=None) == E_NULL and f(r=P + 2) == E_ALIGN
    assert b(dx=None) == E_NULL and b(dg=None) == E_NULL and b(w=None) == E_ARG and b(s=None) == E_ARG and b(w2=None) == E_ARG
    need = lib.ttt_block_norm_partial_bytes(6, 64)
    assert need > 0 and b(bytes=need - 1) == E_WS and b(part=None) == E_WS
    assert lib.ttt_block_norm_partial_bytes(0, 64) == 0 and lib.ttt_block_norm_partial_bytes(6, 8193) == 0


def test_ffn(lib):
    f, b = (lambda **kw: _call(lib.ttt_ffn_fwd, FFN, **kw)), (lambda **kw: _call(lib.ttt_ffn_bwd, FFN_BWD, **kw))
    for c in (f, b):
        for bad in (dict(R=0), dict(D=0), dict(F=0), dict(D=(1 << 20) + 8, ldx=1 << 21), dict(F=(1 << 20) + 1), dict(ldx=63),
                    dict(ldx=65), dict(ldx=(1 << 21) + 8), dict(R=0x7fffffff), dict(R=1 << 30, F=1 << 20)):
            assert c(**bad) == E_SHAPE, bad
        assert c(dtype=3) == E_DTYPE and c(act=0) == E_ARG and c(act=3) == E_ARG
        assert c(x=None) == E_NULL and c(wu=None) == E_NULL and c(x=Q) == E_ALIGN and c(wg=Q) == E_ALIGN and c(bg=P + 1) == E_ALIGN
        assert c(dtype=F32, ws=None) == E_WS and c(D=60, ldx=60, ws=None) == E_WS
    assert f(y=None) == E_NULL and f(R=64, x=Q, y=None) == E_NULL  # few rows may lie anywhere
    assert b(dwg=None) == E_ARG and b(lddy=47) == E_SHAPE and b(dy=None) == E_NULL and b(ws=None) == E_WS and b(ws=Q) == E_ALIGN
    assert lib.ttt_ffn_workspace_bytes(100, 64, 48, BF16) == 0 and lib.ttt_ffn_workspace_bytes(64, 60, 48, F32) == 0
    n = lib.ttt_ffn_workspace_bytes(100, 60, 48, F32)
    assert n > 0 and f(dtype=F32, D=60, bytes=n - 1) == E_WS
    assert b(bytes=lib.ttt_ffn_bwd_workspace_bytes(100, 64, 48, BF16) - 1) == E_WS


def _delta(B=2, L=5, H=4, G=2, N=32, Pd=64, lead=2):
    r = lambda *s: torch.zeros(s[:1] + s[2:] if lead == 1 else s)  # noqa: E731
    return dict(q=r(B, L, G, N), k=r(B, L, G, N), v=r(B, L, H, Pd), g=r(B, L, H), beta=r(B, L, H))


def test_delta_arguments():
    from ttt_amd.delta import gated_delta, gated_delta_step
    ok = _delta()
    with pytest.raises(ValueError, match="GPU"):
        gated_delta(**ok)
    for bad, what in ((dict(v=torch.zeros(2, 5, 4, 48)), "head dim"), (dict(v=torch.zeros(2, 5, 256)), "B,L,H,P"),
                      (dict(q=torch.zeros(2, 5, 2, 16)), "q and k"), (dict(g=torch.zeros(2, 5, 3)), "g must be"),
                      (dict(beta=torch.zeros(2, 5, 4, dtype=torch.float16)), "beta must be in"),
                      (dict(k=torch.zeros(2, 5, 2, 32, dtype=torch.bfloat16)), "v's dtype"),
                      (dict(v=torch.zeros(2, 5, 4, 64, dtype=torch.float64), q=ok["q"].double(), k=ok["k"].double()), "dtype")):
        with pytest.raises(ValueError, match=what):
            gated_delta(**{**ok, **bad})
    for N, G in ((24, 2), (144, 2), (32, 3)):
        d = _delta(N=N, G=G)
        with pytest.raises(ValueError, match="width N|groups"):
            gated_delta(**d)
    d = _delta(lead=1)
    with pytest.raises(ValueError, match="no gradient"):
        gated_delta_step(**d, state=torch.zeros(2, 4, 64, 32, requires_grad=True))
    with pytest.raises(ValueError, match="B,H,P"):
        gated_delta_step(**ok, state=torch.zeros(2, 4, 64, 32))


def test_norm_and_ffn_arguments():
    from ttt_amd.ffn import gated_linear
    from ttt_amd.norm import block_norm
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="GPU"):
        block_norm(x, torch.ones(8))
    for kw, what in ((dict(gate=torch.zeros(3, 7)), "gate"), (dict(gate=x.half()), "gate"), (dict(residual=x.half()), "residual"),
                     (dict(residual=torch.zeros(8)), "residual"), (dict(next_weight=torch.ones(8)), "needs a residual"),
                     (dict(eps=0.0), "eps")):
        with pytest.raises(ValueError, match=what):
            block_norm(x, **kw)
    with pytest.raises(ValueError, match="1 to 8192"):
        block_norm(torch.zeros(2, 8193))
    w = torch.zeros(5, 8)
    with pytest.raises(ValueError, match="GPU"):
        gated_linear(x, w, w)
    for a, kw, what in (((x, w, torch.zeros(4, 8)), {}, "w_gate and w_up"), ((x, torch.zeros(5, 7), torch.zeros(5, 7)), {}, "w_gate"),
                        ((x, w.half(), w), {}, "dtype"), ((x, w, w, torch.zeros(4)), {}, "b_gate"),
                        ((x, w, w), dict(activation="relu"), "activation"), ((x, w[:0], w[:0]), {}, "widths")):
        with pytest.raises(ValueError, match=what):
            gated_linear(*a, **kw)


def test_forward_mode_is_refused(monkeypatch):
    """Tangents are not dropped: each operator raises where one is on its way."""
    import torch.autograd.forward_ad as fw
    from ttt_amd import delta, ffn, norm
    x = torch.zeros(3, 8)
    with fw.dual_level():
        t = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises((NotImplementedError, ValueError)):
            norm.block_norm(t, torch.ones(8))
        with pytest.raises((NotImplementedError, ValueError)):
            ffn.gated_linear(t, torch.zeros(5, 8), torch.zeros(5, 8))
        d = _delta(lead=1)
        d["v"] = fw.make_dual(d["v"], torch.ones_like(d["v"]))
        with pytest.raises(NotImplementedError):
            delta.gated_delta_step(**d, state=torch.zeros(2, 4, 64, 32))


def test_config():
    from ttt_amd.model import ModelConfig
    ok = dict(model_dim=128, num_heads=4, ssm_layer="gated_delta")
    ModelConfig(**ok, seq_len=77, mini_batch_size=13)  # which are the other layers'
    for bad in (dict(state_dim=24), dict(state_dim=144), dict(num_groups=3), dict(conv_width=5), dict(num_layers=0),
                dict(ffn_dim=-1), dict(model_dim=192)):
        with pytest.raises(ValueError):
            ModelConfig(**{**ok, **bad})
