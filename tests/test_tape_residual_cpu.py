"""CPU-only: a residual stream through the tape's norm with addition.  The norm's backward is handed the gradient that the stream already has, adds it in its own
launch and writes the sum to a tensor of its own, since the other addend of the next layer shares that gradient."""
import pytest
import torch

from wav2sleep_amd import generic, lib


def norm(r, w, eps):
    return r * torch.rsqrt(r.pow(2).mean(-1, keepdim=True) + eps) * w


@pytest.mark.parametrize('layers', [1, 2, 3])
def test_the_norm_adds_the_streams_gradient(monkeypatch, layers):
    calls = []

    def fwd(x, w, y, eps, res=None, r=None, rstd=None):   # the kernel's statement in plain torch operations
        s = x if res is None else x + res
        if res is not None:
            r.copy_(s)
        y.copy_(norm(s, w, eps))

    def bwd(r, w, rstd, gy, gr, gx, gw, eps):
        calls.append((gr is not None, gx is gr))
        with torch.enable_grad():
            a, b = r.detach().requires_grad_(True), w.detach().requires_grad_(True)
            ga, gb = torch.autograd.grad(norm(a, b, eps), (a, b), gy)
        gx.copy_(ga if gr is None else ga + gr)
        gw.copy_(gb)
    monkeypatch.setattr(lib, 'add_norm_fwd', fwd)
    monkeypatch.setattr(lib, 'add_norm_bwd', bwd)
    sums = []
    gf = generic.GenericForward(grad=True)
    gf._add = lambda a, b: sums.append(1) or a + b
    g = torch.Generator().manual_seed(layers)
    x, w = torch.randn(5, 16, generator=g, dtype=torch.float64), [torch.nn.Parameter(torch.randn(16, generator=g, dtype=torch.float64)) for _ in range(layers + 1)]
    monkeypatch.setattr(torch.Tensor, 'float', lambda t: t)   # (the tape's gradients are fp32 on the device; here all is 64 bits)
    gx, g_out = [], torch.randn(5, 16, generator=g, dtype=torch.float64)
    keep = g_out.clone()
    with torch.no_grad():
        root, h, res = torch.zeros(1), x, None
        gf._rec(x, (root,), lambda v: (gx.append(v.clone()) or None,))
        for k in range(layers):
            n, res = gf._add_norm(h, res, w[k], 1e-5)
            h = 2.0 * n * n.abs()
            gf._rec(h, (n,), lambda v, n=n: (4.0 * n.abs() * v,))
        out, _ = gf._add_norm(h, res, w[layers], 1e-5)
        got = gf.backward(out, g_out)
    xs, h, res = x.clone().requires_grad_(True), None, None
    ws = [p.detach().requires_grad_(True) for p in w]
    h = xs
    for k in range(layers):
        res = h if res is None else h + res
        n = norm(res, ws[k], 1e-5)
        h = 2.0 * n * n.abs()
    want = torch.autograd.grad(norm(h + res, ws[layers], 1e-5), [xs, *ws], g_out)
    # some 50 roundings of 2^-53 a layer on sums of 16 that may cancel: far below 1e-9
    assert torch.allclose(gx[0], want[0], rtol=1e-9, atol=1e-9)
    assert all(torch.allclose(got[p], v, rtol=1e-9, atol=1e-9) for p, v in zip(w, want[1:]))
    assert calls == [(False, False)] + [(True, False)] * layers and not sums
    assert torch.equal(g_out, keep)
