"""The gated delta-rule stack and the forecaster on it: against the same model in plain float64
operations, forward and gradients; a prompt and single tokens; a step in a graph."""

import pytest
import torch
import torch.nn.functional as Fn

from oracle import block_oracle as O
from oracle import ssm_oracle as S

pytestmark = pytest.mark.gpu


def config(**kw):
    from ttt_amd.model import ModelConfig
    return ModelConfig(**{**dict(model_dim=128, num_heads=4, ssm_layer="gated_delta", state_dim=32, num_groups=2,
                                 num_layers=2, ffn_dim=200), **kw})


def plain(model, x):
    """The forecaster's output in float64 on the CPU, of its own parameters"""
    from ttt_amd.model import GatedDelta
    p = lambda t: t.double()  # noqa: E731
    lin = lambda m, t: t @ p(m.weight).T + (0 if m.bias is None else p(m.bias))  # noqa: E731
    stack = model.ttt.ttt
    r = lin(model.in_proj, x)
    y = O.block_norm(r, p(stack.first_norm))
    for i, part in enumerate(stack.parts):
        if isinstance(part, GatedDelta):
            D, C, H, n = part.width, part.conv_channels, part.num_heads, part.groups * part.state_dim
            z, qkv, b, dt = lin(part.in_proj, y).split([D, C, H, H], -1)
            qkv, _ = S.causal_conv(qkv, p(part.conv_weight), p(part.conv_bias), None, "silu")
            q, k, v = qkv.split([n, n, D], -1)
            g = -torch.exp(p(part.A_log)) * Fn.softplus(dt + p(part.dt_bias))
            o, _ = O.gated_delta(q.unflatten(-1, (part.groups, -1)), k.unflatten(-1, (part.groups, -1)),
                                 v.unflatten(-1, (H, -1)), g, torch.sigmoid(b))
            y = lin(part.wo, O.block_norm(o, p(part.norm_weight), gate=z.unflatten(-1, (H, -1))).flatten(-2))
        else:
            y = lin(part.down, O.gated_linear(y, p(part.w_gate), p(part.w_up)))
        r, y = O.block_norm(y, p(stack.out_norms[i]), r, None, p(stack.scales[i]), p(stack.next_norms[i]))
    return lin(model.head, y[:, -1]).view(len(x), model.pred_len, model.d_out)


@pytest.mark.parametrize("kw", [{}, dict(num_layers=1, ffn_dim=0), dict(num_layers=1, model_dim=192, num_heads=3,
                                                                       num_groups=1, state_dim=64)])
def test_forecaster(lib, kw):
    """Within 1e-4 of float64 in fp32 (some thousand roundings of 2^-24 on the way through two
    blocks, whose parts and norms keep a relative error within some times), gradients within 1e-3."""
    from ttt_amd.model import TTTForecaster
    torch.manual_seed(1)
    model = TTTForecaster(config(**kw), d_in=7, d_out=7, pred_len=6)
    x, dy = torch.randn(3, 70, 7), torch.randn(3, 6, 7)
    params = list(model.parameters())
    want = plain(model, x.double())
    gw = torch.autograd.grad(want, params, dy.double())
    gpu = TTTForecaster(config(**kw), d_in=7, d_out=7, pred_len=6)
    gpu.load_state_dict(model.state_dict())
    gpu.cuda()
    got = gpu(x.cuda())
    assert float((got.double().cpu() - want).norm() / want.norm()) < 1e-4
    gg = torch.autograd.grad(got, list(gpu.parameters()), dy.cuda())
    total = torch.cat([g.flatten() for g in gw]).norm()
    for (n, _), a, b in zip(gpu.named_parameters(), gg, gw):
        off = float((a.double().cpu() - b).norm())
        assert off < 1e-3 * max(float(b.norm()), 1e-4 * float(total)), n


def test_last_token_alone_and_single_tokens(lib):
    """The last token's output is that of all tokens', and a prompt goes on token by token."""
    from ttt_amd.model import TTTForecaster
    torch.manual_seed(2)
    model = TTTForecaster(config(), d_in=7, d_out=7, pred_len=6).cuda().eval()
    x = torch.randn(2, 90, 7, device="cuda")
    with torch.no_grad():
        h = model.in_proj(x)
        torch.testing.assert_close(model.ttt(h, last_only=True), model.ttt(h)[:, -1], rtol=1e-4, atol=1e-5)
        want = [model(x[:, :t + 1]) for t in range(80, 90)]
        y, cache = model.prompt(x[:, :50])
        y, cache = model.prompt(x[:, 50:81], cache)
        torch.testing.assert_close(y, want[0], rtol=1e-3, atol=1e-4)
        for t in range(81, 90):
            torch.testing.assert_close(model.step(x[:, t], cache), want[t - 80], rtol=1e-3, atol=1e-4)


def test_step_in_a_graph(lib):
    from ttt_amd.model import TTTForecaster
    torch.manual_seed(3)
    model = TTTForecaster(config(), d_in=7, d_out=7, pred_len=6).cuda().eval()
    x = torch.randn(4, 40, 7, device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
        _, a = model.prompt(x[:, :30])
        _, b = model.prompt(x[:, :30])
        token = x[:, 30].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _, warm = model.prompt(x[:, :30])
            model.step(token, warm)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = model.step(token, a)
        for t in range(30, 40):
            token.copy_(x[:, t])
            g.replay()
            want = model.step(x[:, t], b)
            torch.cuda.synchronize()
            assert torch.equal(y, want), t


def test_trains_under_autocast(lib):
    """Every parameter has a finite gradient, in bf16."""
    from ttt_amd.model import TTTForecaster
    torch.manual_seed(4)
    model = TTTForecaster(config(), d_in=7, d_out=7, pred_len=6).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = model(torch.randn(4, 130, 7, device="cuda")).float().square().mean()
    loss.backward()
    for n, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), n
