"""Forward-mode derivatives of the state-space operators are refused, as the framework's
other operators refuse them, and not dropped (no GPU: the launches are replaced)."""

import pytest
import torch
from torch.autograd import forward_ad

from tests._stubs import launches  # noqa: F401

B, L, H, P, G, N = 2, 5, 2, 32, 1, 16


def _conv(t):
    from ttt_amd.ssm import causal_conv
    return causal_conv(t["x"], t["w"], t["b"], t["s"], "silu")


def _conv_step(t):
    from ttt_amd.ssm import causal_conv_step
    return causal_conv_step(t["x"], t["s"], t["w"], t["b"])


def _scan(t):
    from ttt_amd.ssm import selective_scan
    return selective_scan(t["x"], t["dt"], t["A"], t["Bm"], t["Cm"], t["D"], t["bias"], t["h"])


def _scan_step(t):
    from ttt_amd.ssm import selective_scan_step
    return selective_scan_step(t["x"], t["dt"], t["A"], t["Bm"], t["Cm"], t["h"], t["D"], t["bias"])


def _norm(t):
    from ttt_amd.norm import layer_norm
    return layer_norm(t["x"], t["w"], t["b"], t["z"])


r = torch.randn
CALLS = {
    "conv": (_conv, lambda: dict(x=r(B, L, 8), w=r(8, 4), b=r(8), s=r(B, 3, 8))),
    "conv step": (_conv_step, lambda: dict(x=r(B, 8), w=r(8, 4), b=r(8), s=r(B, 3, 8))),
    "scan": (_scan, lambda: dict(x=r(B, L, H, P), dt=r(B, L, H), A=-torch.rand(H), Bm=r(B, L, G, N), Cm=r(B, L, G, N), D=r(H),
                                 bias=r(H), h=r(B, H, P, N))),
    "scan step": (_scan_step, lambda: dict(x=r(B, H, P), dt=r(B, H), A=-torch.rand(H), Bm=r(B, G, N), Cm=r(B, G, N), D=r(H),
                                           bias=r(H), h=r(B, H, P, N))),
    "norm": (_norm, lambda: dict(x=r(B, 8), w=r(8), b=r(8), z=r(B, 8)))}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(launches, name, grad):  # noqa: F811
    call, inputs = CALLS[name]
    for k in inputs():
        t = inputs()
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            t[k] = forward_ad.make_dual(t[k], torch.ones_like(t[k]))
            with pytest.raises(NotImplementedError):
                call(t)


@pytest.mark.parametrize("name", CALLS)
def test_calls_without_a_tangent_run(launches, name):  # noqa: F811
    """Within a level too, where no input has one."""
    call, inputs = CALLS[name]
    with forward_ad.dual_level(), torch.no_grad():
        call(inputs())
    assert launches.calls


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms_are_refused(launches, name):  # noqa: F811
    call, inputs = CALLS[name]
    t = inputs()
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: call({**t, "x": x}), (t["x"],), (torch.ones_like(t["x"]),))
