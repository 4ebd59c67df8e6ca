"""Forward-mode derivatives of a gated delta-rule block's operators are refused, by each for a tangent of
each of its inputs, and not dropped (no GPU: the launches are replaced)."""

import contextlib

import pytest
import torch
from torch.autograd import forward_ad

from tests._stubs import launches  # noqa: F401

B, L, H, P, G, N = 2, 5, 2, 32, 1, 16


@pytest.fixture(autouse=True)
def no_gpu(launches, monkeypatch):  # noqa: F811
    from ttt_amd import delta, ffn
    for m in (delta, ffn):
        monkeypatch.setattr(m, "check_device", lambda *ts: ts[0].device)
        monkeypatch.setattr(m, "on_device", lambda dev: contextlib.nullcontext())
        monkeypatch.setattr(m, "_stream", lambda dev: 0)
    return launches


def _delta(t):
    from ttt_amd.delta import gated_delta
    return gated_delta(t["q"], t["k"], t["v"], t["g"], t["beta"], t["state"], return_final_state=True)


def _delta_step(t):
    from ttt_amd.delta import gated_delta_step
    return gated_delta_step(t["q"], t["k"], t["v"], t["g"], t["beta"], t["state"])


def _norm(t):
    from ttt_amd.norm import block_norm
    return block_norm(t["x"], t["w"], t["res"], t["z"], t["s"], t["w2"])


def _ffn(t):
    from ttt_amd.ffn import gated_linear
    return gated_linear(t["x"], t["wg"], t["wu"], t["bg"], t["bu"])


r = torch.randn
CALLS = {
    "delta": (_delta, lambda: dict(q=r(B, L, G, N), k=r(B, L, G, N), v=r(B, L, H, P), g=-torch.rand(B, L, H), beta=torch.rand(B, L, H),
                                   state=r(B, H, P, N))),
    "delta step": (_delta_step, lambda: dict(q=r(B, G, N), k=r(B, G, N), v=r(B, H, P), g=-torch.rand(B, H), beta=torch.rand(B, H),
                                             state=r(B, H, P, N))),
    "norm": (_norm, lambda: dict(x=r(B, 8), w=r(8), res=r(B, 8), z=r(B, 8), s=r(8), w2=r(8))),
    "ffn": (_ffn, lambda: dict(x=r(B, 8), wg=r(5, 8), wu=r(5, 8), bg=r(5), bu=r(5)))}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(no_gpu, name, grad):
    call, inputs = CALLS[name]
    for k in inputs():
        t = inputs()
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            t[k] = forward_ad.make_dual(t[k], torch.ones_like(t[k]))
            with pytest.raises(NotImplementedError):
                call(t)


@pytest.mark.parametrize("name", CALLS)
def test_calls_without_a_tangent_run(no_gpu, name):
    """Within a level too, where no input has one."""
    call, inputs = CALLS[name]
    with forward_ad.dual_level(), torch.no_grad():
        call(inputs())
    assert no_gpu.calls


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms_are_refused(no_gpu, name):
    call, inputs = CALLS[name]
    t = inputs()
    first = next(iter(t))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: call({**t, first: x}), (t[first],), (torch.ones_like(t[first]),))
