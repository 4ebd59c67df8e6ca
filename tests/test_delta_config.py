"""Which heads and widths ModelConfig takes for the gated delta-rule stack: those of its operators."""

import pytest


@pytest.mark.parametrize("heads,dim", [(4, 32), (4, 64), (2, 96), (3, 128), (1, 256), (32, 256), (128, 64)])
def test_widths_of_the_stack(heads, dim):
    from ttt_amd.model import ModelConfig, TTTWrapper
    cfg = ModelConfig(model_dim=heads * dim, num_heads=heads, ssm_layer="gated_delta", seq_len=9)
    if heads * dim <= 512:
        layer = TTTWrapper(cfg).ttt
        assert layer.parts[0].head_dim == dim


@pytest.mark.parametrize("heads,dim,what", [(4, 48, "multiple of 32"), (4, 16, "multiple of 32"), (2, 288, "multiple of 32"),
                                            (33, 256, "8192"), (129, 64, "8192")])
def test_widths_that_are_refused(heads, dim, what):
    from ttt_amd.model import ModelConfig
    with pytest.raises(ValueError, match=what):
        ModelConfig(model_dim=heads * dim, num_heads=heads, ssm_layer="gated_delta")


@pytest.mark.parametrize("layer", ["ttt_linear", "ttt_mlp", "selective_scan"])
def test_the_other_layers_keep_theirs(layer):
    from ttt_amd.model import ModelConfig
    for kw in (dict(model_dim=192, num_heads=2), dict(model_dim=256, num_heads=2), dict(model_dim=1088, num_heads=17)):
        with pytest.raises(ValueError):
            ModelConfig(**kw, ssm_layer=layer)
