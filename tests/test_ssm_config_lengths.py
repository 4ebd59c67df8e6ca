"""The selective state-space layer has no mini-batches: its configuration asks nothing of
them (no GPU)."""

import pytest


@pytest.mark.parametrize("seq_len,K", [(100, 64), (1, 64), (777, 16), (384, 64), (96, 8), (96, 128)])
def test_any_length(seq_len, K):
    from ttt_amd.model import ModelConfig, TTTWrapper
    cfg = ModelConfig(seq_len=seq_len, mini_batch_size=K, ssm_layer="selective_scan", model_dim=128)
    m = TTTWrapper(cfg)
    assert m.rope.shape[0] == cfg.compressed_num_frames == seq_len


@pytest.mark.parametrize("layer", ["ttt_linear", "ttt_mlp"])
def test_the_other_layers_still_ask(layer):
    from ttt_amd.model import ModelConfig
    for bad in (dict(seq_len=100), dict(seq_len=96, mini_batch_size=8), dict(seq_len=256, mini_batch_size=128),
                dict(seq_len=80, mini_batch_size=40)):
        with pytest.raises(ValueError):
            ModelConfig(ssm_layer=layer, **bad)
    ModelConfig(ssm_layer=layer, seq_len=96, mini_batch_size=48)
