"""The gated delta-rule stack's forecaster with heads that only this layer takes, against the same model
in plain float64 operations, and a prompt that goes on token by token."""

import pytest
import torch

from tests.test_gpu_delta_layer import config, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,kw", [(2, 96, {}), (3, 128, dict(num_groups=3, state_dim=48)), (1, 256, dict(num_groups=1)),
                                          (9, 128, dict(num_layers=1, num_groups=3, state_dim=64))])
def test_forecaster(lib, heads, dim, kw):
    """Within 1e-4 of float64 in fp32, gradients within 1e-3, as with heads of 32 and 64."""
    from ttt_amd.model import TTTForecaster
    kw = {**dict(model_dim=heads * dim, num_heads=heads), **kw}
    torch.manual_seed(1)
    model = TTTForecaster(config(**kw), d_in=7, d_out=7, pred_len=6)
    x, dy = torch.randn(2, 70, 7), torch.randn(2, 6, 7)
    want = plain(model, x.double())
    gw = torch.autograd.grad(want, list(model.parameters()), dy.double())
    want = want.detach()
    gpu = TTTForecaster(config(**kw), d_in=7, d_out=7, pred_len=6)
    gpu.load_state_dict(model.state_dict())
    gpu.cuda()
    got = gpu(x.cuda())
    assert float((got.detach().double().cpu() - want).norm() / want.norm()) < 1e-4
    gg = torch.autograd.grad(got, list(gpu.parameters()), dy.cuda())
    total = torch.cat([g.flatten() for g in gw]).norm()
    for (n, _), a, b in zip(gpu.named_parameters(), gg, gw):
        off = float((a.double().cpu() - b).norm())
        assert off < 1e-3 * max(float(b.norm()), 1e-4 * float(total)), n
    with torch.no_grad():
        _, cache = gpu.prompt(x[:, :69].cuda())
        torch.testing.assert_close(gpu.step(x[:, 69].cuda(), cache), got.detach(), rtol=1e-3, atol=1e-4)
