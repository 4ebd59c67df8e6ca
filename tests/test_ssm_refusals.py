"""What the state-space operators refuse, without a GPU: the C entry points return
their status before any launch, the Python ones raise."""

import ctypes

import pytest
import torch

OK, E_SHAPE, E_DTYPE, E_NULL, E_ALIGN, E_HIP, E_WS, E_ARG = 0, -1, -2, -3, -4, -5, -6, -7
F32, BF16, F16 = 0, 1, 2
P, Q = 0x10000, 0x10008  # aligned and misaligned addresses, never read


@pytest.fixture(scope="module")
def lib():
    from ttt_amd import _lib
    return _lib.load()


def _call(fn, defaults, **kw):
    a = dict(defaults)
    assert set(kw) <= set(a), set(kw) - set(a)
    a.update(kw)
    return fn(*a.values())


CONV = dict(x=P, ldx=64, state=P, w=P, bias=P, B=2, L=9, C=64, W=4, act=1, dtype=BF16, y=P, last=P, stream=None)
CONV_BWD = dict(x=P, ldx=64, state=P, w=P, bias=P, dy=P, dlast=P, B=2, L=9, C=64, W=4, act=1, dtype=BF16, dx=P, ds=P,
                dw=P, db=P, part=P, bytes=1 << 30, stream=None)
CONV_STEP = dict(x=P, ldx=64, state=P, w=P, bias=P, B=2, C=64, W=4, act=1, dtype=BF16, y=P, stream=None)
SCAN_IN = dict(x=P, ldx=256, dt=P, ldt=4, A=P, b=P, ldb=128, c=P, ldc=128, D=P, bias=P)
DIMS = dict(B=2, L=99, H=4, P=64, G=2, N=64, dtype=BF16, dtd=BF16, softplus=1)
SCAN = dict(**SCAN_IN, h0=P, **DIMS, y=P, last=P, states=P, sbytes=1 << 40, ws=P, wbytes=1 << 40, stream=None)
SCAN_BWD = dict(**SCAN_IN, dy=P, ldy=256, dlast=P, states=P, sbytes=1 << 40, **DIMS, dx=P, ddt=P, dA=P, dB=P, dC=P, dD=P,
                dbias=P, dh0=P, ws=P, wbytes=1 << 40, stream=None)
SCAN_STEP = dict(**SCAN_IN, h=P, B=2, H=4, P=64, G=2, N=64, dtype=BF16, dtd=BF16, softplus=1, y=P, stream=None)
NORM = dict(x=P, ldx=64, gate=P, ldg=64, w=P, b=P, R=5, D=64, eps=1e-6, dtype=BF16, y=P, stats=P, stream=None)
NORM_BWD = dict(x=P, ldx=64, gate=P, ldg=64, w=P, stats=P, dy=P, R=5, D=64, dtype=BF16, dx=P, dg=P, dw=P, db=P, part=P,
                bytes=1 << 30, stream=None)


def test_conv(lib):
    f, b, s = (lambda fn, d: lambda **kw: _call(fn, d, **kw))(lib.ttt_causal_conv_fwd, CONV), \
        (lambda **kw: _call(lib.ttt_causal_conv_bwd, CONV_BWD, **kw)), \
        (lambda **kw: _call(lib.ttt_causal_conv_step, CONV_STEP, **kw))
    for g in (f, b, s):
        assert g(W=1) == E_SHAPE and g(W=5) == E_SHAPE
        assert g(B=0) == E_SHAPE and g(C=0) == E_SHAPE and g(ldx=63) == E_SHAPE
        assert g(dtype=3) == E_DTYPE and g(act=2) == E_ARG
        assert g(x=None) == E_NULL and g(w=None) == E_NULL and g(x=P + 1) == E_ALIGN and g(w=P + 2) == E_ALIGN
    assert f(L=0) == E_SHAPE and f(L=0x7fffffff) == E_SHAPE and f(y=None) == E_NULL
    assert s(state=None) == E_NULL
    for g in (f, b, s):
        assert g(C=(1 << 22) + 1, ldx=1 << 23) == E_SHAPE
    assert f(B=1 << 20, L=1 << 20) == E_SHAPE and b(B=1 << 20, L=1 << 20) == E_SHAPE
    need = lib.ttt_causal_conv_partial_bytes(2, 9, 64, 4)
    assert need > 0 and lib.ttt_causal_conv_partial_bytes(2, 9, 64, 5) == 0
    assert b(bytes=need - 1) == E_WS and b(part=None) == E_WS and b(part=Q) == E_ALIGN and b(dx=None) == E_NULL


def test_scan(lib):
    f, b, s = (lambda **kw: _call(lib.ttt_scan_fwd, SCAN, **kw)), (lambda **kw: _call(lib.ttt_scan_bwd, SCAN_BWD, **kw)), \
        (lambda **kw: _call(lib.ttt_scan_step, SCAN_STEP, **kw))
    for g in (f, b, s):
        for bad in (dict(P=48), dict(P=128, ldx=512), dict(N=8), dict(N=72, ldb=144, ldc=144), dict(N=144, ldb=288, ldc=288),
                    dict(G=3), dict(G=0), dict(H=0), dict(B=0), dict(ldx=255), dict(ldb=120), dict(ldt=3)):
            assert g(**bad) == E_SHAPE, bad
        assert g(dtype=3) == E_DTYPE and g(dtd=F16) == E_DTYPE
        assert g(x=None) == E_NULL and g(A=None) == E_NULL and g(c=None) == E_NULL
        assert g(A=P + 2) == E_ALIGN and g(dt=P + 1) == E_ALIGN
    for g in (f, b):
        assert g(L=0) == E_SHAPE and g(ldx=260) == E_SHAPE  # rows off 16 bytes
        assert g(x=Q) == E_ALIGN and g(b=Q) == E_ALIGN
        # rows of a chunk beyond 32-bit offsets, where there is more than one
        assert g(ldx=1 << 25) == E_SHAPE and g(ldb=1 << 25) == E_SHAPE and g(ldc=1 << 25) == E_SHAPE
        assert g(ldx=1 << 25, L=1, A=None) == E_NULL
        assert g(H=1 << 18, ldx=1 << 24) == E_SHAPE and g(B=1 << 24) == E_SHAPE  # too many for a grid
    assert b(ldy=1 << 25) == E_SHAPE
    assert s(B=1 << 23) == E_SHAPE
    assert s(b=P + 4) == E_ALIGN and s(ldb=130) == E_SHAPE and s(h=None) == E_NULL and s(h=Q) == E_ALIGN
    assert f(y=None) == E_NULL and f(h0=Q) == E_ALIGN
    need = lib.ttt_scan_states_bytes(2, 99, 4, 64, 64, BF16)
    assert need == 2 * 4 * 2 * 64 * 64 * 4  # a state for each chunk of 64 tokens
    assert lib.ttt_scan_states_bytes(2, 99, 4, 64, 64, F32) == 2 * 4 * 4 * 64 * 64 * 4  # of 32
    assert lib.ttt_scan_states_bytes(2, 99, 4, 48, 64, BF16) == 0
    assert f(sbytes=need - 1) == E_WS and b(sbytes=need - 1) == E_WS and b(states=None) == E_WS
    ws = lib.ttt_scan_workspace_bytes(2, 99, 4, 64, 64, BF16)
    assert ws > 0 and f(wbytes=ws - 1) == E_WS and f(ws=None) == E_WS
    assert lib.ttt_scan_workspace_bytes(64, 99, 12, 64, 64, BF16) == 0  # sequences and heads enough
    wb = lib.ttt_scan_bwd_workspace_bytes(2, 99, 4, 64, 2, 64, BF16)
    assert b(wbytes=wb - 1) == E_WS and b(ws=None) == E_WS and b(ws=Q) == E_ALIGN
    assert lib.ttt_scan_bwd_workspace_bytes(2, 99, 4, 64, 3, 64, BF16) == 0


def test_norm(lib):
    f, b = (lambda **kw: _call(lib.ttt_layer_norm_fwd, NORM, **kw)), (lambda **kw: _call(lib.ttt_layer_norm_bwd, NORM_BWD, **kw))
    for g in (f, b):
        assert g(D=0) == E_SHAPE and g(D=16385, ldx=16385, ldg=16385) == E_SHAPE and g(R=0) == E_SHAPE
        assert g(R=1 << 31) == E_SHAPE and g(ldx=63) == E_SHAPE and g(ldg=63) == E_SHAPE
        assert g(dtype=9) == E_DTYPE and g(x=None) == E_NULL and g(x=P + 1) == E_ALIGN
    assert f(eps=0.0) == E_ARG and f(eps=float("nan")) == E_ARG and f(w=None) == E_NULL and f(y=None) == E_NULL
    assert b(dw=None) == E_NULL and b(dg=None) == E_NULL and b(gate=None) == E_NULL
    need = lib.ttt_layer_norm_partial_bytes(5, 64)
    assert need > 0 and b(bytes=need - 1) == E_WS and b(part=None) == E_WS


def test_python_refusals():
    """Shapes, types and options, before the device is asked for."""
    from ttt_amd.norm import layer_norm
    from ttt_amd.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    z = torch.zeros
    ok = dict(x=z(2, 5, 4, 64), dt=z(2, 5, 4), A=z(4), Bm=z(2, 5, 2, 32), Cm=z(2, 5, 2, 32))
    for bad in (dict(x=z(2, 5, 4, 48)), dict(x=z(2, 5, 256)), dict(Bm=z(2, 5, 3, 32), Cm=z(2, 5, 3, 32)),
                dict(Bm=z(2, 5, 2, 24), Cm=z(2, 5, 2, 24)), dict(Bm=z(2, 5, 2, 144), Cm=z(2, 5, 2, 144)),
                dict(Cm=z(2, 5, 2, 16)), dict(Bm=z(2, 4, 2, 32), Cm=z(2, 4, 2, 32)), dict(dt=z(2, 5, 3)),
                dict(Bm=z(2, 5, 2, 32).half()), dict(dt=z(2, 5, 4).half()),
                ):
        with pytest.raises(ValueError):
            selective_scan(**{**ok, **bad})
    with pytest.raises(ValueError, match="GPU"):
        selective_scan(**ok)
    with pytest.raises(ValueError, match="activation"):
        causal_conv(z(1, 4, 8), z(8, 4), activation="relu")
    for w in (z(8, 1), z(8, 5), z(7, 4), z(8)):
        with pytest.raises(ValueError):
            causal_conv(z(1, 4, 8), w)
    with pytest.raises(ValueError, match="GPU"):
        causal_conv(z(1, 4, 8), z(8, 4))
    with pytest.raises(ValueError, match="no gradient"):
        causal_conv_step(z(1, 8).requires_grad_(True), z(1, 3, 8), z(8, 4))
    with pytest.raises(ValueError, match="no gradient"):
        selective_scan_step(z(2, 4, 64), z(2, 4), z(4).requires_grad_(True), z(2, 2, 32), z(2, 2, 32), z(2, 4, 64, 32))
    for bad in (dict(weight=z(8)), dict(gate=z(3, 7)), dict(gate=z(3, 8).half()), dict(eps=0.0),
                ):
        with pytest.raises(ValueError):
            layer_norm(z(3, 8), **bad)
    with pytest.raises(ValueError):
        layer_norm(z(1, 16385))
    with pytest.raises(ValueError, match="GPU"):
        layer_norm(z(3, 8))


def test_a_library_error_names_the_call(lib):
    from ttt_amd import _lib
    with pytest.raises(ValueError, match="ttt_scan_fwd"):
        _lib.check(_call(lib.ttt_scan_fwd, SCAN, N=8), "ttt_scan_fwd")
    assert ctypes.sizeof(ctypes.c_longlong) == 8
