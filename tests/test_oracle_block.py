"""The plain forms of a gated delta-rule block against themselves another way: the delta rule's
written-out gradients against autograd of its forward and against differences, and against its
states multiplied out."""

import pytest
import torch

from oracle import block_oracle as O


def _args(seed, B=2, L=6, H=4, G=2, N=5, P=3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    return ([r(B, L, G, N), r(B, L, G, N), r(B, L, H, P), -torch.rand(B, L, H, generator=g, dtype=torch.float64),
             torch.rand(B, L, H, generator=g, dtype=torch.float64), r(B, H, P, N)], r(B, L, H, P), r(B, H, P, N))


@pytest.mark.parametrize("unit", [True, False])
def test_delta_gradients(unit):
    args, do, dl = _args(1)
    if not unit:
        args[1] = O._unit(args[1])
    for t in args:
        t.requires_grad_(True)
    o, h = O.gated_delta(*args, unit=unit)
    want = torch.autograd.grad([o, h], args, [do, dl])
    got = O.gated_delta_all(*(t.detach() for t in args), do, dl, unit=unit)
    torch.testing.assert_close(got["o"], o.detach(), rtol=1e-12, atol=1e-12)
    for k, w in zip(("q", "k", "v", "g", "beta", "state"), want):
        torch.testing.assert_close(got["d" + k], w, rtol=1e-10, atol=1e-10)
    assert torch.autograd.gradcheck(lambda *a: O.gated_delta(*a, unit=unit), args, eps=1e-6, atol=1e-6)


def test_delta_state_as_products():
    """S_t = a S_{t-1} (1 - b k k^T) + b v k^T"""
    (q, k, v, g, b, s), _, _ = _args(2, H=2, G=2)
    ku = O._unit(k)
    want = s
    for t in range(k.shape[1]):
        kk = ku[:, t, :, :, None] * ku[:, t, :, None, :]
        eye = torch.eye(k.shape[-1], dtype=k.dtype)
        want = torch.exp(g[:, t])[..., None, None] * want @ (eye - b[:, t, :, None, None] * kk) + \
            (b[:, t, :, None] * v[:, t])[..., None] * ku[:, t, :, None, :]
    torch.testing.assert_close(O.gated_delta(q, k, v, g, b, s)[1], want, rtol=1e-12, atol=1e-12)


def test_sizes_bound_the_values():
    args, do, dl = _args(3)
    v, s = (O.gated_delta_all(*args, do, dl, sizes=q) for q in (False, True))
    for k in v:
        assert (v[k].abs() <= s[k] * (1 + 1e-12)).all(), k


def test_norms_and_projections_differences():
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    f = lambda *a: O.block_norm(*a)  # noqa: E731
    assert torch.autograd.gradcheck(f, [r(3, 5), r(5), r(3, 5), r(3, 5), r(5), r(5)], eps=1e-6, atol=1e-6)
    for act in ("silu", "gelu"):
        assert torch.autograd.gradcheck(lambda *a: O.gated_linear(*a, activation=act),
                                        [r(3, 4), r(6, 4), r(6, 4), r(6), r(6)], eps=1e-6, atol=1e-6)
