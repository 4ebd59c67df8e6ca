"""The selective state-space layer's configuration and parameters (no GPU)."""

import pytest
import torch


def test_config_refuses_what_the_kernels_do_not_take():
    from ttt_amd.model import ModelConfig
    ok = dict(ssm_layer="selective_scan", model_dim=256, num_heads=4, mini_batch_size=16)
    ModelConfig(**ok)
    ModelConfig(**ok, state_dim=128, num_groups=4, conv_width=2)
    for bad in (dict(state_dim=8), dict(state_dim=72), dict(state_dim=144), dict(num_groups=3), dict(num_groups=0),
                dict(conv_width=1), dict(conv_width=5), dict(num_heads=2)):
        with pytest.raises(ValueError):
            ModelConfig(**{**ok, **bad})
    ModelConfig(ssm_layer="ttt_linear", model_dim=128, state_dim=8)  # the other layers do not read it


def test_parameters():
    from ttt_amd.model import ModelConfig, SelectiveSSM, TTTWrapper
    torch.manual_seed(0)
    m = TTTWrapper(ModelConfig(ssm_layer="selective_scan", model_dim=256, num_heads=4, mini_batch_size=16, num_groups=2,
                               state_dim=32))
    assert isinstance(m.ttt, SelectiveSSM)
    shapes = {n: tuple(p.shape) for n, p in m.ttt.named_parameters()}
    C = 256 + 2 * 2 * 32
    assert shapes == {"conv_weight": (C, 4), "conv_bias": (C,), "A_log": (4,), "D": (4,), "dt_bias": (4,),
                      "in_proj.weight": (256 + C + 4, 256), "in_proj.bias": (256 + C + 4,), "post_norm.weight": (256,),
                      "post_norm.bias": (256,), "wo.weight": (256, 256), "wo.bias": (256,)}
    assert set(m.state_dict()) == {"ttt." + n for n in shapes}
    rates, steps = torch.exp(m.ttt.A_log), torch.nn.functional.softplus(m.ttt.dt_bias)
    assert (rates >= 1).all() and (rates <= 16).all() and (steps >= 9.9e-4).all() and (steps <= 0.101).all()
    with pytest.raises(ValueError, match="GPU"):
        m(torch.zeros(1, 3, 256))
