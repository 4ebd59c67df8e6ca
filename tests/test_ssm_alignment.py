"""States and their gradients that begin off 16 bytes are copied, not refused (no GPU: the
launches are replaced)."""

import pytest
import torch

from tests._stubs import launches, rows_at  # noqa: F401


def _off(shape, by):
    """Contiguous fp32 values that begin `by` elements behind 16 bytes"""
    n = torch.Size(shape).numel()
    t = torch.randn(n + 8)
    first = -(t.data_ptr() // 4) % 4 + by
    t = t[first:first + n].view(shape)
    assert t.is_contiguous() and t.data_ptr() % 16 == 4 * by
    return t


@pytest.mark.parametrize("by", [0, 1, 2, 3])
def test_scan_states(launches, by):  # noqa: F811
    from ttt_amd.ssm import selective_scan
    B, L, H, P, G, N = 2, 5, 3, 32, 1, 16
    h0, dlast = _off((B, H, P, N), by), _off((B, H, P, N), by)
    x = torch.randn(B, L, H, P, requires_grad=True)
    seen = []

    def look(at, want):
        def f(*a):
            assert a[at] % 16 == 0
            assert torch.equal(rows_at(a[at], want.numel(), 1, want.numel(), want.dtype)[0], want.flatten())
            seen.append((a[at] == want.data_ptr()) == (by == 0))  # and where they lie right, read in place
        return f

    launches.look["ttt_scan_fwd"], launches.look["ttt_scan_bwd"] = look(11, h0), look(13, dlast)
    y, last = selective_scan(x, torch.randn(B, L, H), -torch.rand(H), *(torch.randn(B, L, G, N) for _ in range(2)),
                             initial_state=h0, return_final_state=True)
    torch.autograd.grad([y, last], x, [torch.randn_like(y), dlast])
    assert seen == [True, True]
