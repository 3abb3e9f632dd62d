"""The host side of the state space mixer's operators: what torch may hand them beside plain tensors."""
import pytest
import torch
import torch.fx.experimental.proxy_tensor
from torch.autograd import forward_ad

import wav2sleep_amd as W
from tests.test_mixer_ops_gpu import rnd

pytestmark = pytest.mark.gpu


def calls(B=2, L=6, D=8, N=4, K=4):
    """name -> (function, keyword tensors): every operator with all of its tensors"""
    x, w, b = rnd(1, B, L, D), rnd(2, D, K), rnd(3, D)
    scan = dict(u=x, dt=rnd(4, B, L, D), A=-rnd(5, D, N).abs(), B=rnd(6, B, L, N), C=rnd(7, B, L, N), D=rnd(8, D), z=rnd(9, B, L, D), dt_bias=rnd(10, D), state=rnd(11, B, D, N))
    row = {k: (v[:, 0].contiguous() if v.dim() == 3 and k != 'state' else v) for k, v in scan.items()}
    conv = dict(x=x, weight=w, bias=b, state=rnd(12, B, K - 1, D))
    norm = dict(x=x, weight=b, residual=rnd(13, B, L, D))
    return dict(short_conv=(W.short_conv, conv), short_conv_step=(W.short_conv_step, dict(conv, x=x[:, 0].contiguous(), state_out=rnd(14, B, K - 1, D))),
                ssm_scan=(W.ssm_scan, scan), ssm_step=(W.ssm_step, dict(row, state_out=rnd(15, B, D, N))),
                add_rms_norm=(W.add_rms_norm, norm), add_rms_norm_8bit=(W.add_rms_norm_8bit, norm))


OPERATORS = ['short_conv', 'short_conv_step', 'ssm_scan', 'ssm_step', 'add_rms_norm', 'add_rms_norm_8bit']


@pytest.mark.parametrize('name', OPERATORS)
def test_forward_mode_is_refused(name):
    """no kernel carries a tangent on: whichever argument has one, the call raises, and steps leave their state as it was"""
    f, kw = calls()[name]
    for k, v in kw.items():
        kept = {n: t.clone() for n, t in kw.items()}
        with forward_ad.dual_level():
            with pytest.raises(W.lib.W2SError, match='forward-mode'):
                f(**{**kw, k: forward_ad.make_dual(v, torch.ones_like(v))})
            f(**{**kept, k: forward_ad.unpack_dual(forward_ad.make_dual(kept[k], torch.ones_like(v))).primal})
        assert all(torch.equal(kw[n], kept[n]) for n in kw if 'state_out' not in kw or n != 'state_out')
    f(**kw)


def test_forward_mode_through_the_mixer_is_refused():
    m, x = W.SequenceSSM(64, num_layers=1).to('cuda').eval(), rnd(1, 2, 3, 64)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: m(d), lambda: m.prompt(d), lambda: m.step(forward_ad.make_dual(x[:, 0].contiguous(), torch.ones_like(x[:, 0])), m.init_state(2))):
            with pytest.raises(W.lib.W2SError, match='forward-mode'):
                call()
    assert torch.isfinite(m(x)).all()


@pytest.mark.parametrize('name', ['short_conv', 'ssm_scan', 'add_rms_norm'])
def test_forward_mode_over_a_gradient_is_refused(name):
    f, kw = calls()[name]
    x = kw['u' if name == 'ssm_scan' else 'x'].requires_grad_(True)
    y = f(**kw)
    y = y[0] if isinstance(y, tuple) else y
    gy = torch.ones_like(y)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch.autograd.grad(y, x, forward_ad.make_dual(gy, gy), retain_graph=True)
    assert torch.isfinite(torch.autograd.grad(y, x, gy)[0]).all()


@pytest.mark.parametrize('name', OPERATORS)
def test_negative_views_and_zeros_without_memory(name):
    """a real tensor may stand for the negative of what lies in memory (a part of a conjugate), or for zeros that lie nowhere"""
    run = lambda kw: [t for t in (lambda o: o if isinstance(o, tuple) else (o,))(f(**kw))] + [kw[k] for k in kw if k == 'state_out']   # noqa: E731
    f, kw = calls()[name]
    fresh = lambda: {k: v.clone() for k, v in kw.items()}   # noqa: E731
    for k, v in kw.items():
        if k == 'state_out' or (k == 'state' and 'state_out' in kw):   # a step's states have to lie in memory
            for odd in (torch._neg_view(v.clone()), torch._efficientzerotensor(v.shape, device='cuda')):
                with pytest.raises(W.lib.W2SError):
                    f(**{**fresh(), k: odd})
            continue
        want = run(fresh())
        for a, b in zip(run({**fresh(), k: torch._neg_view(-v)}), want):
            assert torch.equal(a.float(), b.float()), k
        for a, b in zip(run({**fresh(), k: torch._efficientzerotensor(v.shape, device='cuda')}), run({**fresh(), k: torch.zeros_like(v)})):
            assert torch.equal(a.float(), b.float()), k


@pytest.mark.parametrize('name', ['short_conv', 'ssm_scan', 'add_rms_norm'])
def test_gradients_of_and_through_negative_views(name):
    f, kw = calls()[name]
    first = lambda o: o[0] if isinstance(o, tuple) else o   # noqa: E731

    def grads(odd):
        leaves = {k: v.clone().requires_grad_(True) for k, v in kw.items()}
        y = first(f(**{k: (torch._neg_view(-v) if odd else v) for k, v in leaves.items()}))
        gy = rnd(30, *y.shape)
        return torch.autograd.grad(y, list(leaves.values()), torch._neg_view(-gy) if odd else gy)
    for k, a, b in zip(kw, grads(True), grads(False)):
        assert torch.equal(a, b), k


def test_a_conjugates_imaginary_part_of_one_channel():
    c = torch.complex(rnd(1, 2, 6, 1), rnd(2, 2, 6, 1))
    x, w = c.conj().imag, rnd(3, 1, 4)
    assert x.is_neg() and torch.equal(W.short_conv(x, w), W.short_conv(x.clone(), w))


@pytest.mark.filterwarnings('ignore')
@pytest.mark.parametrize('name', OPERATORS)
def test_a_trace_is_refused(name):
    """a trace records dispatched operators only: it would hold the allocation of the result and not the launch that fills it"""
    f, kw = calls()[name]
    first = next(iter(kw))
    out = lambda o: o[0].float() if isinstance(o, tuple) else o   # noqa: E731
    with pytest.raises(W.lib.W2SError, match='trace'):
        torch.jit.trace(lambda t: out(f(**{**kw, first: t})), (kw[first],), check_trace=False)
    with pytest.raises(W.lib.W2SError, match='trace'):
        torch.fx.experimental.proxy_tensor.make_fx(lambda t: out(f(**{**kw, first: t})))(kw[first])
    f(**kw)


def test_a_compiled_caller_runs_them_as_they_are():
    """no trace: a compiler leaves the call in the program, also with gradients, and other dispatch modes go on around it"""
    from torch.utils.flop_counter import FlopCounterMode
    f, kw = calls()['short_conv']
    x = kw['x'].clone().requires_grad_(True)
    run = lambda t: (f(**{**kw, 'x': 2 * t}) + 1).sum()   # noqa: E731
    want = torch.autograd.grad(run(x), x)[0]
    assert torch.equal(torch.autograd.grad(torch.compile(run, backend='aot_eager')(x), x)[0], want)
    with FlopCounterMode(display=False):
        assert torch.equal(torch.autograd.grad(run(x), x)[0], want)
