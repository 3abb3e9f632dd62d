"""CPU-only checks of the state space sequence mixer: construction, its place in the model's config tree, refusals."""
import pytest
import torch

import wav2sleep_amd as W


def _model():
    return W.Wav2Sleep(W.SignalEncoders({'THX': 'THX'}, 64, 'gelu', norm='instance', chunk_causal=False, max_channels=32), W.MultiModalAttentionEmbedder(64, layers=1, nhead=4, dim_ff=64),
                       W.SequenceSSM(64, num_layers=2, state_dim=8, expand=1), 4)


def test_config_tree_rebuilds_the_model(tmp_path):
    from wav2sleep_amd.checkpoint import save_model
    m = _model()
    assert not m.fused_ok() and m.config_dict()['sequence_mixer']['_target_'] == 'wav2sleep_amd.SequenceSSM'
    save_model(str(tmp_path), m)
    back = W.load_model(str(tmp_path), device='cpu')
    assert all(torch.equal(a, b) for a, b in zip(m.state_dict().values(), back.state_dict().values()))
    assert back.sequence_mixer.config_dict() == m.sequence_mixer.config_dict()


def test_refusals():
    for kw in (dict(feature_dim=100), dict(dt_rank=8), dict(state_dim=12), dict(state_dim=72), dict(kernel_size=9)):
        with pytest.raises(ValueError):
            W.SequenceSSM(**{**dict(feature_dim=64), **kw})
    m = W.SequenceSSM(64, num_layers=1)
    with pytest.raises(W.lib.W2SError):
        m(torch.zeros(1, 3, 64))
    with pytest.raises(W.lib.W2SError):
        m.step(torch.zeros(1, 64), m.init_state(1))
    with pytest.raises(ValueError):
        m.step(torch.zeros(1, 32), m.init_state(1))
    with pytest.raises(ValueError):
        m.step(torch.zeros(1, 64), [])


def test_refusals_of_a_prompt():
    m = W.SequenceSSM(64, num_layers=1)
    with pytest.raises(ValueError):
        m.prompt(torch.zeros(1, 0, 64))
    with pytest.raises(ValueError):
        m.prompt(torch.zeros(1, 3, 64), state=[])
    with pytest.raises(W.lib.W2SError):
        m.prompt(torch.zeros(1, 3, 64))
