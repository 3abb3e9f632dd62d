"""Plain 64-bit statements of the state space mixer's operators and of their gradients, position by position, for the tests.

Every function also takes `mag=True`: the same formula with every term's absolute value, i.e. how large the sums are that a result is the
(possibly cancelled) outcome of.  An fp32 evaluation of a sum of terms is off by at most (number of roundings on a term's way) x 2^-24 x that."""
import torch

U32 = 2.0 ** -24   # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, mag, roundings, what=''):
    """|got - want| <= half a step of got's type x |want| (its one rounding; half its smallest number near zero) + roundings x 2^-24 x mag"""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    dt = got.dtype
    g = got.detach().double()
    assert torch.isfinite(g).all(), f'{what}: not finite'
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    tol = half_step(dt) * (want.abs() + roundings * U32 * mag) + roundings * U32 * mag + tiny
    off = (g - want).abs() - tol
    at = int(off.argmax())
    assert float(off.max()) <= 0.0, (f'{what}: worst at flat index {at} of {tuple(got.shape)}: got {float(g.reshape(-1)[at])}, want {float(want.reshape(-1)[at])}, '
                                     f'tolerance {float(tol.reshape(-1)[at])}')


def d64(t):
    return None if t is None else t.detach().double()


def alive(lengths, B, L, device):
    if lengths is None:
        return torch.ones(B, L, dtype=torch.bool, device=device)
    return torch.arange(L, device=device)[None] < lengths.long().clamp(0, L)[:, None]


def _silu(x):
    s = torch.sigmoid(x)
    return x * s, s * (1 + x * (1 - s))


def scan(u, dt, A, Bm, Cm, D=None, z=None, bias=None, softplus=True, state=None, lengths=None, gy=None, gs=None, mag=False):
    """-> dict(y, last[, gu, gdt, gA, gB, gC, gD, gz, gbias, gstate])"""
    u, dt, A, Bm, Cm, D, z, bias, state, gy, gs = (d64(t) for t in (u, dt, A, Bm, Cm, D, z, bias, state, gy, gs))
    m = torch.abs if mag else (lambda t: t)
    B, L, Dc = u.shape
    N, G = A.shape[1], Bm.shape[2]
    dev = u.device
    on = alive(lengths, B, L, dev)
    clean = lambda t: torch.where(on.reshape(B, L, *[1] * (t.dim() - 2)), t, torch.zeros((), dtype=t.dtype, device=dev))   # noqa: E731
    u, raw, Bm, Cm = m(clean(u)), clean(dt) + (0 if bias is None else bias), m(clean(Bm)), m(clean(Cm))
    each = Dc // G
    Be, Ce = (t.repeat_interleave(each, dim=2) for t in (Bm, Cm))
    delta = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    Dv = torch.zeros(Dc, dtype=torch.float64, device=dev) if D is None else m(D)
    h0 = torch.zeros(B, Dc, N, dtype=torch.float64, device=dev) if state is None else m(state)
    h, hs, a = h0, [], []
    for t in range(L):
        a.append(torch.exp(delta[:, t, :, None] * A))
        new = a[t] * h + m((delta[:, t] * u[:, t])[..., None]) * Be[:, t]
        h = torch.where(on[:, t, None, None], new, h)
        hs.append(h)
    last = h
    H = torch.stack(hs, 1) if L else u.new_zeros(B, 0, Dc, N)
    pre = (Ce * H).sum(-1) + Dv * u
    if z is None:
        gate, gslope = torch.ones_like(u), torch.zeros_like(u)
    else:
        gate, gslope = (m(t) for t in _silu(clean(z)))
    out = dict(y=clean(pre * gate), last=last)
    if gy is None and gs is None:
        return out
    gy = m(clean(gy)) if gy is not None else torch.zeros_like(u)
    gp = gy * gate
    e = m(gs) if gs is not None else torch.zeros_like(h0)
    out.update(gA=torch.zeros_like(A), gu=torch.zeros_like(u), gdt=torch.zeros_like(u), gB=torch.zeros_like(Be), gC=torch.zeros_like(Ce))
    for t in range(L - 1, -1, -1):
        k = on[:, t, None, None]
        g = torch.where(k, Ce[:, t] * gp[:, t, :, None] + e, torch.zeros_like(e))
        prev = hs[t - 1] if t else h0
        eh = g * a[t] * prev
        d = m(delta[:, t])
        out['gA'] += (eh * d[..., None]).sum(0)
        sB = (g * Be[:, t]).sum(-1)
        out['gdt'][:, t] = ((eh * m(A)).sum(-1) + u[:, t] * sB) * slope[:, t]
        out['gu'][:, t] = d * sB + Dv * gp[:, t]
        out['gB'][:, t] = g * (d * u[:, t])[..., None]
        out['gC'][:, t] = torch.where(k, gp[:, t, :, None] * hs[t], torch.zeros_like(g))
        e = torch.where(k, g * a[t], e)
    out['gB'], out['gC'] = (out[q].unflatten(2, (G, each)).sum(3) for q in ('gB', 'gC'))
    out.update(gD=(gp * u).sum((0, 1)), gbias=out['gdt'].sum((0, 1)), gz=gy * pre * gslope, gstate=e)
    return out


def conv(x, w, b=None, silu=True, state=None, lengths=None, gy=None, gs=None, mag=False):
    """-> dict(y, last[, gx, gw, gb, gstate])"""
    x, w, b, state, gy, gs = (d64(t) for t in (x, w, b, state, gy, gs))
    m = torch.abs if mag else (lambda t: t)
    B, L, D = x.shape
    K = w.shape[1]
    on = alive(lengths, B, L, x.device)[..., None]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    x = torch.where(on, x, zero)
    n = torch.full((B,), L, device=x.device) if lengths is None else lengths.long().clamp(0, L)
    full = torch.cat([x.new_zeros(B, K - 1, D) if state is None else state, x], 1)
    bias = 0 if b is None else b
    z = sum(full[:, k:k + L] * w[:, k] for k in range(K)) + bias
    act, slope = _silu(z) if silu else (z, torch.ones_like(z))
    if mag:   # |silu(z)| <= |z| and it moves by at most 1.1 times what z does: the size of z's own sum; the slope is at most 1.1
        act, slope = sum(full[:, k:k + L].abs() * w[:, k].abs() for k in range(K)) + (0 if b is None else b.abs()), torch.full_like(z, 1.1)
    at = n[:, None] + torch.arange(K - 1, device=x.device)[None]
    last = torch.gather(full, 1, at[..., None].expand(-1, -1, D))
    out = dict(y=torch.where(on, act, zero), last=last)
    if gy is None and gs is None:
        return out
    gz = torch.where(on, m(gy) * slope, zero) if gy is not None else torch.zeros_like(x)
    gf = torch.zeros_like(full)
    for k in range(K):
        gf[:, k:k + L] += gz * m(w[:, k])
    if gs is not None:
        for bi in range(B):
            for j in range(K - 1):
                gf[bi, int(at[bi, j])] += m(gs[bi, j])
    out.update(gx=torch.where(on, gf[:, K - 1:], zero), gstate=gf[:, :K - 1], gb=gz.sum((0, 1)),
               gw=torch.stack([(gz * m(full[:, k:k + L])).sum((0, 1)) for k in range(K)], 1))
    return out


def norm(x, w, res=None, eps=1e-5, gy=None, gr=None, mag=False):
    """-> dict(y, r[, g, gw])"""
    x, w, res, gy, gr = (d64(t) for t in (x, w, res, gy, gr))
    m = torch.abs if mag else (lambda t: t)
    r = x if res is None else x + res
    size = m(x) if res is None else m(x) + m(res)   # (a cancelled sum is off by its addends' size)
    rstd = 1 / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + eps)
    n = size * rstd
    out = dict(y=n * m(w), r=size)
    if gy is None and gr is None:
        return out
    gy = m(gy) if gy is not None else torch.zeros_like(r)
    gn = gy * m(w)
    back = n * (gn * n).mean(-1, keepdim=True)
    g = rstd * (gn + back if mag else gn - back)
    if gr is not None:
        g = g + m(gr)
    out.update(g=g, gw=(gy * n).reshape(-1, n.shape[-1]).sum(0))
    return out
