"""What the backwards of the state-space operators read where saved tensors come back in
another layout than they were saved in (no GPU: the launches are replaced)."""

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

from tests._stubs import launches, rows_at  # noqa: F401


class Layout:
    """Hooks that give every saved tensor back in another layout, and remember what they gave."""

    def __init__(self, how):
        self.how, self.given = how, {}

    def unpack(self, t):
        if self.how == "contiguous":
            r = t.clone(memory_format=torch.contiguous_format)
        elif self.how == "transposed":
            r = t.transpose(0, -1).contiguous().transpose(0, -1)
        elif self.how == "odd address":
            flat = torch.empty(t.numel() + 1, dtype=t.dtype)[1:]
            r = flat.view(t.shape).copy_(t)
        else:  # columns of a matrix that is wider than the one before
            wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 56, dtype=t.dtype)
            r = wide[..., 8:8 + t.shape[-1]].copy_(t)
        self.given[r.data_ptr()] = r
        return r

    def __enter__(self):
        self.hooks = saved_tensors_hooks(lambda t: t, self.unpack)
        self.hooks.__enter__()
        return self

    def __exit__(self, *e):
        return self.hooks.__exit__(*e)

    def rows(self, address, ld, want, lead):
        """Rows from `address` on, `ld` apart, are `want` [.., width], and stay inside what is there."""
        want = want.flatten(lead).flatten(0, lead - 1)
        n, width = want.shape
        if address in self.given:
            t = self.given[address]
            t = t.flatten(lead) if t.dim() > lead + 1 else t
            assert ld == t.stride(lead - 1), "rows of the tensor that came back, at the stride of another"
        else:
            assert ld == width, "rows of a copy"
        assert torch.equal(rows_at(address, ld, n, width, want.dtype), want)


HOWS = ["contiguous", "transposed", "odd address", "wider"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("how", HOWS)
def test_conv(launches, how, dt):  # noqa: F811
    from ttt_amd.ssm import causal_conv
    B, L, C, W = 2, 7, 32, 4
    x = torch.randn(B, L, 100).to(dt)[..., 4:4 + C]
    w, b, s = torch.randn(C, W), torch.randn(C), torch.randn(B, W - 1, C).to(dt)
    leaves = [t.requires_grad_(True) for t in (x.detach(), w, b, s)]
    seen = []

    def bwd(xp, ldx, sp, wp, bp, *rest):
        m.rows(xp, ldx, x, 2)
        for p, t in ((sp, s), (wp, w), (bp, b)):
            assert torch.equal(rows_at(p, t.numel(), 1, t.numel(), t.dtype)[0], t.detach().flatten())
        seen.append(ldx)

    launches.look["ttt_causal_conv_bwd"] = bwd
    with Layout(how) as m:
        y, last = causal_conv(*leaves, activation="silu", return_final_state=True)
    torch.autograd.grad([y, last], leaves, [torch.randn_like(y), torch.randn_like(last)])
    assert seen


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("how", HOWS)
def test_scan(launches, how, dt):  # noqa: F811
    from ttt_amd.ssm import selective_scan
    B, L, H, P, G, N = 2, 9, 2, 32, 2, 16
    xbc = torch.randn(B, L, 24 + H * P + 2 * G * N).to(dt)[..., 24:]
    x = xbc[..., :H * P].unflatten(-1, (H, P))
    Bm, Cm = (xbc[..., H * P + k * G * N:H * P + (k + 1) * G * N].unflatten(-1, (G, N)) for k in (0, 1))
    step = torch.randn(B, L, H + 5).to(dt)[..., 3:3 + H]
    par = [-torch.rand(H), torch.randn(H), torch.randn(H)]
    leaves = [t.detach().requires_grad_(True) for t in (x, step, par[0], Bm, Cm, par[1], par[2])]
    seen = []

    def bwd(xp, ldx, dp, ldd, Ap, bp, ldb, cp, ldc, Dp, biasp, *rest):
        for p, ld, t in ((xp, ldx, x), (dp, ldd, step), (bp, ldb, Bm), (cp, ldc, Cm)):
            m.rows(p, ld, t, 2)
        for p, t in ((Ap, par[0]), (Dp, par[1]), (biasp, par[2])):
            assert torch.equal(rows_at(p, H, 1, H, t.dtype)[0], t)
        for p, ld in ((xp, ldx), (bp, ldb), (cp, ldc)):
            assert p % 16 == 0 and ld * x.element_size() % 16 == 0
        seen.append(ldx)

    launches.look["ttt_scan_bwd"] = bwd
    with Layout(how) as m:
        y = selective_scan(*leaves)
    torch.autograd.grad(y, leaves, torch.randn_like(y))
    assert seen


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("gated", [True, False])
def test_norm(launches, how, dt, gated):  # noqa: F811
    from ttt_amd.norm import layer_norm
    R, D = 6, 40
    x = torch.randn(R, 64).to(dt)[:, 8:8 + D]
    z = torch.randn(R, 100).to(dt)[:, 3:3 + D] if gated else None
    w, b = torch.randn(D), torch.randn(D)
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, z)]
    seen = []

    def bwd(xp, ldx, gp, ldg, wp, *rest):
        m.rows(xp, ldx, x, 1)
        if gated:
            m.rows(gp, ldg, z, 1)
        assert torch.equal(rows_at(wp, D, 1, D, w.dtype)[0], w)
        seen.append(ldx)

    launches.look["ttt_layer_norm_bwd"] = bwd
    with Layout(how) as m:
        y = layer_norm(*leaves)
    torch.autograd.grad(y, [t for t in leaves if t is not None], torch.randn_like(y))
    assert seen
