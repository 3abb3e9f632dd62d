"""`SequenceSSM` of other sizes than the usual ones, through autograd, and with rows behind a night's end that hold anything.  Bars as in test_sequence_ssm_gpu.py
(split-bf16 matrix products: 1e-3 of the largest feature, 2e-3 relative L2 of a gradient)."""
import pytest
import torch

import wav2sleep_amd as W
from tests.test_sequence_ssm_gpu import reference

pytestmark = pytest.mark.gpu
SIZES = [dict(feature_dim=16, num_layers=1, expand=1, state_dim=8, kernel_size=1), dict(feature_dim=48, num_layers=3, expand=3, state_dim=24, kernel_size=8, dt_rank=32),
         dict(feature_dim=128, num_layers=2, expand=2, state_dim=64, kernel_size=2)]


def mixer(seed=0, **kw):
    torch.manual_seed(seed)
    m = W.SequenceSSM(**kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.02 * torch.randn_like(p))
    return m.to('cuda').eval()


@pytest.mark.parametrize('kw', SIZES, ids=str)
def test_sizes(kw):
    from wav2sleep_amd.generic import GenericForward
    m, F = mixer(**kw), kw['feature_dim']
    x, g = torch.randn(2, 37, F, device='cuda'), torch.randn(2, 37, F, device='cuda')
    want, P = reference(m, x)
    grads = dict(zip(P, torch.autograd.grad((want * g.double()).sum(), list(P.values()))))
    want = want.detach()
    size = float(want.abs().max())
    assert float((m(x) - want).abs().max()) <= 1e-3 * size
    y, state = m.prompt(x[:, :30])
    assert float((y - want[:, :30]).abs().max()) <= 1e-3 * size
    for t in range(30, 37):
        assert float((m.step(x[:, t], state) - want[:, t]).abs().max()) <= 1e-3 * size, t
    gf = GenericForward(training=True, seed=1, grad=True)
    with torch.no_grad():
        got = gf.backward(gf.sequence_ssm(m, x), g)
    for k, p in m.named_parameters():
        assert float((got[p].double() - grads[k]).norm() / grads[k].norm()) <= 2e-3, k


def test_rows_behind_the_end_may_hold_anything():
    m = mixer(**SIZES[1])
    x = torch.randn(3, 20, 48, device='cuda')
    n = torch.tensor([20, 0, 11], device='cuda', dtype=torch.int32)
    bad = x.clone()
    bad[1], bad[2, 11:] = float('nan'), float('inf')
    (a, sa), (b, sb) = m.prompt(x, lengths=n), m.prompt(bad, lengths=n)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2, :11], b[2, :11])
    for p, q in zip(sa, sb):
        assert all(torch.equal(s, t) for s, t in zip(p, q))
    assert not any(t[1].any() for pair in sa for t in pair)   # a night without epochs: the state in front of it


def test_autograd_through_the_model():
    """model(x) with a gradient is one node: its gradients are the train step's"""
    torch.manual_seed(0)
    enc = W.SignalEncoders({'THX': 'THX'}, 64, 'gelu', norm='instance', chunk_causal=False, max_channels=32)
    model = W.Wav2Sleep(enc, W.MultiModalAttentionEmbedder(64, layers=1, nhead=4, dim_ff=64, dropout=0.0), W.SequenceSSM(64, num_layers=2, state_dim=8, expand=1), 4).to('cuda').train()
    x, y = {'THX': torch.randn(2, 256 * 6, device='cuda')}, torch.randint(0, 4, (2, 6), device='cuda')
    torch.nn.functional.cross_entropy(model(x).flatten(0, 1), y.flatten()).backward()
    got = {k: p.grad.clone() for k, p in model.named_parameters()}
    mod = W.SleepModule(model, num_classes=4, lr=1e-3, max_norm=0.0)
    mod.trainer.step(x, y.float())
    for k, p in model.named_parameters():
        want = mod.trainer.views[p]
        assert float((got[k] - want).norm()) <= 1e-5 * float(want.norm()) + 1e-9, k   # (two forms of the loss' own gradient, the same launches behind them)


@pytest.mark.filterwarnings('ignore')
def test_a_trace_of_the_mixer_is_refused():
    m, x = mixer(**SIZES[0]), torch.randn(2, 3, 16, device='cuda')
    for f in (m, lambda t: m.prompt(t)[0]):
        with pytest.raises(W.lib.W2SError, match='trace'):
            torch.jit.trace(f, (x,), check_trace=False)
