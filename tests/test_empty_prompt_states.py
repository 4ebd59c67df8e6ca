"""The state that a call over no tokens hands back is one that a step takes, contiguous, whatever the
strides of the one that it was given (no GPU: the launches are replaced)."""

import contextlib

import pytest
import torch

from tests._stubs import launches  # noqa: F401

B, H, P, G, N = 2, 2, 32, 1, 16


@pytest.mark.parametrize("dt", [torch.float32, torch.float64])
def test_strided_states(launches, monkeypatch, dt):  # noqa: F811
    from ttt_amd import delta, ssm
    monkeypatch.setattr(delta, "check_device", lambda *ts: ts[0].device)
    monkeypatch.setattr(delta, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(delta, "_stream", lambda dev: 0)
    z = lambda *s: torch.zeros(s)  # noqa: E731
    state = torch.randn(B, H, N, P, dtype=dt).transpose(2, 3)
    conv = torch.randn(B, 8, 3, dtype=dt).transpose(1, 2)
    w = z(8, 4)
    _, s = delta.gated_delta(z(B, 0, G, N), z(B, 0, G, N), z(B, 0, H, P), z(B, 0, H), z(B, 0, H), state, return_final_state=True)
    assert s.is_contiguous() and torch.equal(s, state.float()) and s.data_ptr() != state.data_ptr()
    with torch.no_grad():
        delta.gated_delta_step(z(B, G, N), z(B, G, N), z(B, H, P), z(B, H), z(B, H), s)
    _, s = ssm.selective_scan(z(B, 0, H, P), z(B, 0, H), -torch.ones(H), z(B, 0, G, N), z(B, 0, G, N), initial_state=state,
                              return_final_state=True)
    assert s.is_contiguous() and torch.equal(s, state.float())
    with torch.no_grad():
        ssm.selective_scan_step(z(B, H, P), z(B, H), -torch.ones(H), z(B, G, N), z(B, G, N), s)
    _, s = ssm.causal_conv(z(B, 0, 8), w, None, conv, None, True)
    assert s.is_contiguous() and torch.equal(s, conv.float())
    with torch.no_grad():
        ssm.causal_conv_step(z(B, 8), s, w)
    assert [n for n, _ in launches.calls] == ["ttt_delta_step", "ttt_scan_step", "ttt_causal_conv_step"]
