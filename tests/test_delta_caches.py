"""A gated delta-rule stack is handed one cache a block: any other number is refused before a cache is
moved on (no GPU: the check comes before any launch)."""

import pytest
import torch


@pytest.mark.parametrize("blocks", [1, 3])
def test_number_of_caches(blocks):
    from ttt_amd.model import ModelConfig, SSMCache, TTTForecaster, TTTWrapper
    cfg = ModelConfig(model_dim=64, num_heads=2, ssm_layer="gated_delta", state_dim=16, num_layers=blocks, ffn_dim=24)
    stack, model = TTTWrapper(cfg).ttt, TTTForecaster(cfg, d_in=3, d_out=3, pred_len=2)
    cache = lambda: SSMCache(torch.zeros(2, 3, stack.parts[0].conv_channels), torch.zeros(2, 2, 32, 16))  # noqa: E731
    for bad in ([], [cache() for _ in range(blocks - 1)], [cache() for _ in range(blocks + 1)], cache(), [None] * blocks):
        for call in (lambda: stack.step(torch.zeros(2, 64), bad), lambda: stack.prompt(torch.zeros(2, 5, 64), bad),
                     lambda: model.step(torch.zeros(2, 3), bad), lambda: model.prompt(torch.zeros(2, 5, 3), bad)):
            with pytest.raises(ValueError, match=f"list of {blocks} caches"):
                call()
    with pytest.raises(ValueError, match="GPU"):  # (the right number goes on to the operators)
        stack.step(torch.zeros(2, 64), [cache() for _ in range(blocks)])
