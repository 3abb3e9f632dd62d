"""A model with the state space mixer through the training script, its checkpoints and the moving average of its weights."""
import os

import pytest
import torch

import wav2sleep_amd as W
from tests.test_train_mixer_cpu import cli

pytestmark = pytest.mark.gpu


def test_train_script_with_the_mixer(tmp_path, capsys):
    rc = cli().main(['--synthetic', '6', '--synthetic-epochs', '24', '--batch-size', '2', '--epochs', '2', '--signals', 'ECG,THX', '--sequence-mixer', 'ssm', '--out', str(tmp_path / 'run')])
    assert rc == 0 and 'epoch 1: train loss' in capsys.readouterr().out
    model = W.load_model(str(tmp_path / 'run' / 'model'), device='cuda')
    assert isinstance(model.sequence_mixer, W.SequenceSSM)
    x = {'ECG': torch.randn(1, 24 * 1024, device='cuda'), 'THX': torch.randn(1, 24 * 256, device='cuda')}
    with torch.no_grad():
        want = model(x)
    assert tuple(want.shape) == (1, 24, 4)
    mod = W.SleepModule(W.load_model(str(tmp_path / 'run' / 'model'), device='cuda'), num_classes=4)   # resume: the checkpoint holds the weights of the folder
    with torch.no_grad():
        for p in mod.model.parameters():
            p.zero_()
    W.load_lightning_checkpoint(os.path.join(tmp_path, 'run', 'last.ckpt'), mod)
    assert mod.trainer.step_count == 6
    mod.model.eval()
    with torch.no_grad():
        assert torch.equal(mod.model(x), want)


def test_moving_average_of_its_weights():
    torch.manual_seed(0)
    enc = W.SignalEncoders({'THX': 'THX'}, 64, 'gelu', norm='instance', chunk_causal=False, max_channels=32)
    model = W.Wav2Sleep(enc, W.MultiModalAttentionEmbedder(64, layers=1, nhead=4, dim_ff=64), W.SequenceSSM(64, num_layers=2, state_dim=8, expand=1), 4).to('cuda')
    mod = W.SleepModule(model, num_classes=4, lr=1e-3)
    ema = W.EMACallback(decay=0.5)
    ema.setup(pl_module=mod)
    batch = {'THX': torch.randn(2, 256 * 6, device='cuda')}, torch.randint(0, 4, (2, 6), device='cuda').float()
    want = {k: p.detach().clone() for k, p in model.named_parameters()}
    for _ in range(3):
        mod.training_step(batch)
        ema.on_train_batch_end(pl_module=mod)
        want = {k: 0.5 * want[k] + 0.5 * p.detach() for k, p in model.named_parameters()}
    got = ema.state_dict()['ema_state_dict']
    # three rounds of two products and a sum: 9 half steps of fp32 at the most, of values that do not cancel (both of the same weight)
    for k, v in want.items():
        assert float((got['model.' + k] - v).abs().max()) <= 9 * 2.0 ** -24 * float(v.abs().max()) + 1e-30, k
