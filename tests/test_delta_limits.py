"""The sizes that the gated delta rule takes, by the threads of its launches (no GPU: the C entry points
return their status, and the size functions 0, before any launch)."""

import pytest
import torch

from tests._stubs import launches  # noqa: F401
from tests.test_block_refusals import BF16, DELTA, DELTA_BWD, E_NULL, E_SHAPE, F32, _call

CHUNK = {BF16: 64, F32: 32}


@pytest.fixture(scope="module")
def lib():
    from ttt_amd import _lib
    return _lib.load()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H", [(1, 16), (8, 2), (3, 5)])
def test_chunks(lib, dtype, B, H):
    """Fewer than 2^32 threads in a launch: 256 to a chunk and head forwards, 512 in the backward and in a
    forward that it follows."""
    fwd, train = (((1 << 32) - 1) // n // (B * H) * CHUNK[dtype] for n in (256, 512))
    kw = dict(B=B, H=H, G=H, P=32, N=16, dtype=dtype, ldq=16 * H, ldk=16 * H, ldv=32 * H, ldg=H, ldb=H, bd=F32)
    for L, alone, trains in ((train, True, True), (train + 1, True, False), (fwd, True, False), (fwd + 1, False, False)):
        dims = (B, L, H, 32, 16, dtype)
        assert (lib.ttt_delta_workspace_bytes(*dims) > 0) == alone, L
        assert (lib.ttt_delta_saved_bytes(*dims) > 0) == trains, L
        assert (lib.ttt_delta_bwd_workspace_bytes(B, L, H, 32, H, 16, dtype) > 0) == trains, L
        # (a call that is taken goes on to its missing tensor)
        assert _call(lib.ttt_delta_fwd, DELTA, **kw, L=L, saved=None, v=None) == (E_NULL if alone else E_SHAPE), L
        assert _call(lib.ttt_delta_fwd, DELTA, **kw, L=L, v=None) == (E_NULL if trains else E_SHAPE), L
        bwd = {k: v for k, v in kw.items() if k != "ldv"}
        assert _call(lib.ttt_delta_bwd, DELTA_BWD, **bwd, L=L, lddo=32 * H, dq=None) == (E_NULL if trains else E_SHAPE), L


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sums_of_the_heads_that_share(lib, dtype):
    """Their launch has a thread for four values of dq and of dk: B L G N / 2 of them, below 2^32, where heads share
    q and k; each has its own in the call that has as many groups as heads."""
    for G in (8, 4):
        H, most = 2 * G, ((1 << 32) - 256) * 2 // 128 // G
        kw = dict(B=1, H=H, G=G, P=32, N=128, dtype=dtype, ldq=128 * G, ldk=128 * G, ldv=32 * H, ldg=H, ldb=H, bd=F32, v=None)
        for n, ok in ((most, True), (most + 1, False)):
            assert (lib.ttt_delta_bwd_workspace_bytes(1, n, H, 32, G, 128, dtype) > 0) == ok, (G, n)
            assert _call(lib.ttt_delta_fwd, DELTA, **kw, L=n) == (E_NULL if ok else E_SHAPE), (G, n)
        assert _call(lib.ttt_delta_fwd, DELTA, **kw, L=most + 1, saved=None) == E_NULL
    n = ((1 << 32) - 256) * 2 // 128 // 16 + 1
    assert lib.ttt_delta_bwd_workspace_bytes(1, n, 16, 32, 16, 128, dtype) > 0


@pytest.mark.parametrize("train", [True, False])
def test_refused_before_a_launch(launches, monkeypatch, train):  # noqa: F811
    """Where a size function gives 0, the call raises: a forward that trains does not go on without `saved`."""
    from ttt_amd import delta
    monkeypatch.setattr(delta, "check_device", lambda *ts: ts[0].device)
    name = f"ttt_delta_{'saved' if train else 'workspace'}_bytes"
    monkeypatch.setattr(delta, "_bytes", lambda n, *a: 0 if n == name else 1024)
    z = lambda *s: torch.zeros(s, requires_grad=train)  # noqa: E731
    with pytest.raises(ValueError, match="too many"):
        delta.gated_delta(z(1, 3, 1, 16), z(1, 3, 1, 16), z(1, 3, 2, 32), z(1, 3, 2), z(1, 3, 2))
    assert not launches.calls
