"""The plain state-space operators against themselves another way: their written-out
gradients against autograd of their forward, and against differences."""

import pytest
import torch

from oracle import ssm_oracle as S


def _scan_inputs(seed, B=2, L=7, H=4, P=3, G=2, N=5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    return [r(B, L, H, P), r(B, L, H), -torch.rand(H, generator=g, dtype=torch.float64) - 0.1, r(B, L, G, N), r(B, L, G, N),
            r(H), r(H), r(B, H, P, N)], r(B, L, H, P), r(B, H, P, N)


@pytest.mark.parametrize("softplus", [True, False])
def test_scan_gradients(softplus):
    args, dy, dl = _scan_inputs(1)
    if not softplus:
        args[1], args[6] = args[1].abs(), args[6].abs()
    for t in args:
        t.requires_grad_(True)
    y, h = S.selective_scan(*args, softplus=softplus)
    want = torch.autograd.grad([y, h], args, [dy, dl])
    got = S.selective_scan_grads(*(t.detach() for t in args), softplus, dy, dl)
    for k, w in zip(("x", "dt", "A", "Bm", "Cm", "D", "dt_bias", "state"), want):
        torch.testing.assert_close(got[k], w, rtol=1e-10, atol=1e-10)
    assert torch.autograd.gradcheck(lambda *a: S.selective_scan(*a, softplus=softplus), args, eps=1e-6, atol=1e-6)


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("L", [1, 2, 6])
def test_conv_gradients(activation, L):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    args = [r(2, L, 3), r(3, 4), r(3), r(2, 3, 3)]
    dy, dl = r(2, L, 3).detach(), r(2, 3, 3).detach()
    f = lambda x, w, b, s: S.causal_conv(x, w, b, s, activation)  # noqa: E731
    want = torch.autograd.grad(f(*args), args, [dy, dl])
    got = S.causal_conv_grads(*(t.detach() for t in args), activation, dy, dl)
    for k, w in zip(("x", "weight", "bias", "state"), want):
        torch.testing.assert_close(got[k], w, rtol=1e-10, atol=1e-10)
    assert torch.autograd.gradcheck(f, args, eps=1e-6, atol=1e-6)


def test_magnitudes_bound_the_values():
    args, dy, dl = _scan_inputs(3)
    a, m = (S.selective_scan_grads(*args, True, dy, dl, magnitude=q) for q in (False, True))
    for k in a:
        assert (a[k].abs() <= m[k] * (1 + 1e-12)).all(), k
