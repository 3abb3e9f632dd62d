"""The state space mixer's operators (short convolution, selective scan, RMS norm with the residual's addition) against plain 64-bit statements.

Tolerances count roundings (mixer_reference.close): a result may be off by its own rounding and by (roundings on a term's way) x 2^-24 x (the size of
its terms).  The scan: a term of h goes through at most L steps, each of which multiplies it by exp(delta A).  delta carries the softplus' error (its exponential of
|x| <= 12: 12 log2(e) + 1 half steps from the rounded argument and the instruction's own 1 ulp, the series and products 12 more: < 32) and |delta A| <= 3 in
these inputs, so a step costs < 3 x 32 + 8 < 110 half steps at most; ends and sums over N <= 64 states, channels and positions add their own counts."""
import pytest
import torch

import wav2sleep_amd as W
from tests import mixer_reference as R

pytestmark = pytest.mark.gpu
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def rnd(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return torch.randn(*shape, device='cuda', generator=g).to(dtype)


def wide_view(t, off=3):
    """the same values as a slice of a wider tensor: strides and alignment of a projection's part"""
    w = torch.full((*t.shape[:-1], t.shape[-1] + 7), float('nan'), device=t.device, dtype=t.dtype)
    w[..., off:off + t.shape[-1]] = t
    return w[..., off:off + t.shape[-1]]


def lens(kind, B, L):
    if not kind:
        return None
    v = [L, 0, 1, L // 2, max(0, L - 1), L + 5, -3, min(L, 17)]   # clamped on the device
    return torch.tensor([v[i % len(v)] for i in range(B)], device='cuda', dtype=torch.int32)


def poison(t, lengths):
    """NaN behind the end of every sequence"""
    on = R.alive(lengths, t.shape[0], t.shape[1], t.device).reshape(*t.shape[:2], *[1] * (t.dim() - 2))
    return torch.where(on, t, torch.full_like(t, float('nan')))


# ------------------------------------------------------------------------------------------------------------------ scan
def scan_inputs(dtype, B, L, D, N, G, seed=0, gate=True, state=True, ragged=False, extras=True, strided=False):
    dt = DTYPES[dtype]
    p = dict(u=rnd(seed + 1, B, L, D, dtype=dt), dt=(0.7 * rnd(seed + 2, B, L, D) - 3.0).to(dt), Bm=rnd(seed + 3, B, L, G, N, dtype=dt), Cm=rnd(seed + 4, B, L, G, N, dtype=dt),
             A=-(0.1 + 4.0 * torch.rand(D, N, device='cuda', generator=torch.Generator(device='cuda').manual_seed(seed + 5))),
             D=rnd(seed + 6, D) if extras else None, bias=0.3 * rnd(seed + 7, D) if extras else None,
             z=rnd(seed + 8, B, L, D, dtype=dt) if gate else None, state=rnd(seed + 9, B, D, N) if state else None, lengths=lens(ragged, B, L),
             gy=rnd(seed + 10, B, L, D, dtype=dt), gs=rnd(seed + 11, B, D, N) if state else None)
    if ragged:
        for k in ('u', 'dt', 'Bm', 'Cm', 'z', 'gy'):
            if p[k] is not None:
                p[k] = poison(p[k], p['lengths'])
    if strided:
        for k in ('u', 'dt', 'Bm', 'Cm', 'z', 'gy'):
            if p[k] is not None:
                p[k] = wide_view(p[k], off=1 + len(k))
    return p


def reference_scan(p, grads=True, **kw):
    g = dict(gy=p['gy'], gs=p['gs']) if grads else {}
    args = (p['u'], p['dt'], p['A'], p['Bm'], p['Cm'], p['D'], p['z'], p['bias'])
    return [R.scan(*args, state=p['state'], lengths=p['lengths'], mag=m, **g, **kw) for m in (False, True)]


LEAVES = ['u', 'dt', 'A', 'Bm', 'Cm', 'D', 'z', 'bias', 'state']
GRADS = ['gu', 'gdt', 'gA', 'gB', 'gC', 'gD', 'gz', 'gbias', 'gstate']


def check_scan(p, softplus=True):
    B, L, D = p['u'].shape
    N, G = p['A'].shape[1], p['Bm'].shape[2]
    want, mag = reference_scan(p, softplus=softplus)
    q = {k: (v.detach().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}
    kw = dict(D=q['D'], z=q['z'], dt_bias=q['bias'], dt_softplus=softplus, state=q['state'], lengths=q['lengths'])
    step = 110
    fwd = step * (L + 1) + N + 16
    with torch.no_grad():
        y0, last0 = W.ssm_scan(q['u'], q['dt'], q['A'], q['Bm'], q['Cm'], return_state=True, **kw)
        y1 = W.ssm_scan(q['u'], q['dt'], q['A'], q['Bm'], q['Cm'], **kw)
    R.close(y0, want['y'], mag['y'], fwd, 'y')
    R.close(last0, want['last'], mag['last'], fwd, 'state')
    assert torch.equal(y0, y1)
    y, last = W.ssm_scan(q['u'], q['dt'], q['A'], q['Bm'], q['Cm'], return_state=True, **kw)
    R.close(y, want['y'], mag['y'], fwd, 'y (training)')
    leaves = [q[k] for k in LEAVES if q[k] is not None]
    outs, gouts = ([y, last], [p['gy'], p['gs']]) if p['gs'] is not None else ([y], [p['gy']])
    got = torch.autograd.grad(outs, leaves, gouts, retain_graph=True)
    again = torch.autograd.grad(outs, leaves, gouts)
    both = 2 * fwd + D // G + 64   # the way forward to h, the way back to its gradient, the sum over a group's channels
    for k, gname, g, g2 in zip([k for k in LEAVES if q[k] is not None], [n for k, n in zip(LEAVES, GRADS) if q[k] is not None], got, again):
        more = B * L if k in ('A', 'D', 'bias') else 0
        R.close(g, want[gname], mag[gname], both + more, gname)
        assert torch.equal(g, g2), f'{gname}: two runs differ'


SCAN_SHAPES = [(1, 1, 1, 1, 1), (2, 2, 3, 3, 1), (3, 15, 16, 4, 1), (2, 16, 17, 16, 1), (2, 17, 64, 16, 1), (1, 33, 65, 5, 1), (2, 65, 48, 16, 3), (8, 130, 20, 8, 2),
               (3, 127, 33, 24, 1), (1, 128, 16, 32, 1), (2, 129, 40, 64, 1), (1, 300, 100, 16, 2), (4, 64, 128, 16, 1), (1, 513, 32, 16, 1), (5, 31, 36, 17, 9)]


@pytest.mark.parametrize('shape', SCAN_SHAPES, ids=str)
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_scan_and_gradients(dtype, shape):
    check_scan(scan_inputs(dtype, *shape, seed=11))


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('kind', ['ragged', 'strided', 'both', 'bare', 'no_softplus', 'no_gate'])
@pytest.mark.parametrize('shape', [(8, 70, 24, 16, 2), (8, 129, 16, 4, 1)], ids=str)
def test_scan_forms(dtype, kind, shape):
    p = scan_inputs(dtype, *shape, seed=23, ragged=kind in ('ragged', 'both'), strided=kind in ('strided', 'both'), gate=kind not in ('bare', 'no_gate'),
                    state=kind != 'bare', extras=kind != 'bare')
    if kind == 'no_softplus':
        p['dt'] = (p['dt'].float().abs() * 0.05).to(p['dt'].dtype)   # a negative step would grow without bound
        p['bias'] = p['bias'].abs() * 0.1
    check_scan(p, softplus=kind != 'no_softplus')


def test_scan_long_rows_in_pieces():
    """few rows and a long axis; a call over the whole axis, and calls that hand the state on"""
    p = scan_inputs('f32', 1, 3001, 24, 16, 1, seed=5)
    args = lambda lo, hi: [p[k][:, lo:hi] if k != 'A' else p[k] for k in ('u', 'dt', 'A', 'Bm', 'Cm')]   # noqa: E731
    y, last = W.ssm_scan(*args(0, 3001), D=p['D'], z=p['z'], dt_bias=p['bias'], state=p['state'], return_state=True)
    want, mag = reference_scan(p, grads=False)
    R.close(y, want['y'], mag['y'], 110 * 3002, 'y')
    R.close(last, want['last'], mag['last'], 110 * 3002, 'state')
    st, cuts = p['state'], [0, 1, 700, 701, 2048, 3001]
    for lo, hi in zip(cuts, cuts[1:]):
        yk, st = W.ssm_scan(*args(lo, hi), D=p['D'], z=p['z'][:, lo:hi], dt_bias=p['bias'], state=st, return_state=True)
        R.close(yk, want['y'][:, lo:hi], mag['y'][:, lo:hi], 110 * 3002, f'y[{lo}:{hi}]')
    R.close(st, want['last'], mag['last'], 110 * 3002, 'state by pieces')


def test_scan_long_row_gradients():
    check_scan(scan_inputs('f32', 1, 2050, 16, 16, 1, seed=8))


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('shape', [(8, 1200, 16, 16, 1), (3, 700, 20, 40, 1), (4, 900, 16, 6, 2), (2, 520, 8, 32, 1)], ids=str)
def test_scan_ragged_rows_in_segments(dtype, shape):
    """few workgroups and long sequences, some of which end segments before the last"""
    check_scan(scan_inputs(dtype, *shape, seed=41, ragged=True, strided=True))


def test_scan_far_strides():
    """positions far apart: of a sequence of one they do not matter, and a gradient that arrives so is copied"""
    p = scan_inputs('f32', 2, 6, 8, 4, 1, seed=15)
    flat = torch.zeros(5 * (1 << 22) + 64, device='cuda')
    far = lambda t: flat.as_strided(t.shape, (t.shape[2], 1 << 22, 1)).copy_(t)   # noqa: E731
    one = {k: p[k][:, :1] for k in ('dt', 'Bm', 'Cm')}
    y = W.ssm_scan(far(p['u'][:, :1]), one['dt'], p['A'], one['Bm'], one['Cm'])
    assert torch.equal(y, W.ssm_scan(p['u'][:, :1], one['dt'], p['A'], one['Bm'], one['Cm']))
    u = p['u'].clone().requires_grad_(True)
    y = W.ssm_scan(u, p['dt'], p['A'], p['Bm'], p['Cm'])
    a, = torch.autograd.grad(y, u, p['gy'], retain_graph=True)
    b, = torch.autograd.grad(y, u, far(p['gy']))
    assert torch.equal(a, b)


def test_scan_decay_ends():
    """steps so long that the state is forgotten at once, and so short that nothing is"""
    p = scan_inputs('f32', 2, 40, 16, 16, 1, seed=3)
    p['dt'][:, 7] = 60.0
    p['dt'][:, 8] = -80.0
    p['u'][:, 7] = 1e-3
    want, mag = reference_scan(p, grads=False)
    y = W.ssm_scan(p['u'], p['dt'], p['A'], p['Bm'], p['Cm'], D=p['D'], z=p['z'], dt_bias=p['bias'], state=p['state'])
    R.close(y, want['y'], mag['y'], 110 * 41 + 300, 'y')   # (+ a softplus argument of 80: 116 half steps of its exponential; twice for the product)


def test_scan_against_differences():
    """directional derivatives of the 64-bit forward, by central differences, against the kernels' gradients"""
    p = scan_inputs('f32', 2, 37, 20, 8, 2, seed=31)
    q = {k: (v.detach().requires_grad_(True) if k in LEAVES and v is not None else v) for k, v in p.items()}
    y, last = W.ssm_scan(q['u'], q['dt'], q['A'], q['Bm'], q['Cm'], D=q['D'], z=q['z'], dt_bias=q['bias'], state=q['state'], return_state=True)
    got = torch.autograd.grad([y, last], [q[k] for k in LEAVES], [p['gy'], p['gs']])

    def loss(v):
        o = R.scan(v['u'], v['dt'], v['A'], v['Bm'], v['Cm'], v['D'], v['z'], v['bias'], state=v['state'])
        return float((o['y'] * p['gy'].double()).sum() + (o['last'] * p['gs'].double()).sum())
    for i, (k, g) in enumerate(zip(LEAVES, got)):
        way = rnd(77 + i, *p[k].shape).double()
        eps = 1e-5   # the difference's own error ~ eps^2 x third derivative ~ 1e-10 of the sums, and 1e-16 / eps = 1e-11 of the loss
        up, dn = ({**{n: R.d64(t) if n != 'lengths' else t for n, t in p.items()}, k: p[k].double() + s * eps * way} for s in (1, -1))
        want, have = (loss(up) - loss(dn)) / (2 * eps), float((g.double() * way).sum())
        size = float((g.double() * way).abs().sum())
        assert abs(have - want) <= 1e-4 * size, (k, have, want, size)   # 2 (110 x 38) roundings of 2^-24 = 5e-4 of the worst case, far above what sums of random signs give


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('shape', [(1, 1, 1, 1), (3, 17, 5, 1), (2, 64, 16, 2), (5, 48, 24, 3), (4, 30, 64, 1)], ids=str)
def test_scan_step(dtype, shape):
    B, D, N, G = shape
    p = scan_inputs(dtype, B, 1, D, N, G, seed=41)
    want, mag = reference_scan(p, grads=False)
    row = lambda k: p[k][:, 0]   # noqa: E731
    keep = p['state'].clone()
    out = torch.full_like(keep, float('nan'))
    kw = dict(D=p['D'], z=row('z'), dt_bias=p['bias'])
    y = W.ssm_step(row('u'), row('dt'), p['A'], row('Bm'), row('Cm'), p['state'], state_out=out, **kw)
    assert torch.equal(p['state'], keep)
    y2 = W.ssm_step(wide_view(row('u')), wide_view(row('dt')), p['A'], wide_view(row('Bm')), wide_view(row('Cm')), p['state'], D=p['D'], z=wide_view(row('z')), dt_bias=p['bias'])
    for a in (y, y2):
        R.close(a, want['y'][:, 0], mag['y'][:, 0], 110 * 2 + N, 'y')
    for s in (out, p['state']):
        R.close(s, want['last'], mag['last'], 110 * 2, 'state')


# ------------------------------------------------------------------------------------------------------------------ short convolution
def check_conv(dtype, B, L, D, K, silu=True, state=True, ragged=False, strided=False, seed=0, bias=True):
    dt = DTYPES[dtype]
    x, gy = rnd(seed + 1, B, L, D, dtype=dt), rnd(seed + 2, B, L, D, dtype=dt)
    w, b = rnd(seed + 3, D, K), rnd(seed + 4, D) if bias else None
    st, gs = (rnd(seed + 5, B, K - 1, D, dtype=dt), rnd(seed + 6, B, K - 1, D, dtype=dt)) if state else (None, None)
    n = lens(ragged, B, L)
    if ragged:
        x, gy = poison(x, n), poison(gy, n)
    if strided:
        x, gy = wide_view(x), wide_view(gy, 1)
    want, mag = (R.conv(x, w, b, silu, st, n, gy, gs, mag=m) for m in (False, True))
    act = 'silu' if silu else None
    y0 = W.short_conv(x, w, b, act, state=st, lengths=n)
    # K fused steps and the bias; the SiLU's exponential of |z| <= 20 (29 half steps of its rounded argument, 3 more of division and product)
    fwd = K + 2 + 40
    R.close(y0, want['y'], mag['y'], fwd, 'y')
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, st)]
    y, last = W.short_conv(leaves[0], leaves[1], leaves[2], act, state=leaves[3], lengths=n, return_state=True)
    assert torch.equal(y, y0) and torch.equal(last.double(), want['last'])
    live = [t for t in leaves if t is not None]
    got = torch.autograd.grad((y, last) if state else y, live, (gy, gs) if state else gy)
    names = [k for k, t in zip(('gx', 'gw', 'gb', 'gstate'), leaves) if t is not None]
    for k, g in zip(names, got):
        # the slope s (1 + z (1 - s)) moves by at most 0.5 per unit of z, whose own error is `fwd` half steps of its size |z| <= 25: 13 fwd
        R.close(g, want[k], mag[k], 14 * fwd + K + (B * L if k in ('gw', 'gb') else 0), k)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('shape', [(1, 1, 1, 1), (2, 2, 3, 4), (3, 7, 16, 2), (2, 8, 8, 4), (2, 9, 130, 3), (1, 65, 1024, 4), (4, 33, 40, 8), (2, 100, 257, 5), (3, 16, 12, 6),
                                   (1, 300, 24, 7)], ids=str)
def test_conv_and_gradients(dtype, shape):
    check_conv(dtype, *shape, seed=3)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('kind', ['ragged', 'strided', 'both', 'bare', 'linear'])
def test_conv_forms(dtype, kind):
    for L in (3, 50):
        check_conv(dtype, 8, L, 48, 4, silu=kind != 'linear', state=kind != 'bare', ragged=kind in ('ragged', 'both'), strided=kind in ('strided', 'both'), bias=kind != 'bare', seed=9)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('D,K', [(1, 1), (5, 2), (64, 4), (72, 8)])
def test_conv_step_follows_the_sequence(dtype, D, K):
    B, L = 3, 11
    dt = DTYPES[dtype]
    x, w, b = rnd(1, B, L, D, dtype=dt), rnd(2, D, K), rnd(3, D)
    want, last = W.short_conv(x, w, b, return_state=True)
    st = torch.zeros(B, K - 1, D, device='cuda', dtype=dt)
    for t in range(L):
        out = torch.empty_like(st)
        y = W.short_conv_step(x[:, t], st, w, b, state_out=out)
        y2 = W.short_conv_step(wide_view(x[:, t]), st, w, b)   # in place
        assert torch.equal(st, out) and torch.equal(y, y2)
        assert torch.equal(y, want[:, t])   # the same products in the same order
    assert torch.equal(st, last)


# ------------------------------------------------------------------------------------------------------------------ norm
def check_norm(dtype, rows, C, res='same', strided=False, seed=0, scale=1.0):
    dt = DTYPES[dtype]
    rt = torch.float32 if res == 'f32' else dt
    x, w = (scale * rnd(seed + 1, *rows, C)).to(dt), rnd(seed + 2, C)
    r = (scale * rnd(seed + 3, *rows, C)).to(rt) if res else None
    gy, gr = rnd(seed + 4, *rows, C, dtype=dt), rnd(seed + 5, *rows, C, dtype=rt) if res else None
    if strided:
        x, gy = wide_view(x), wide_view(gy, 2)
        r, gr = (wide_view(r, 5), wide_view(gr, 1)) if res else (r, gr)
    want, mag = (R.norm(x, w, r, 1e-5, gy, gr, mag=m) for m in (False, True))
    y0, s0 = W.add_rms_norm(x, w, r)
    # rstd: a sum of C squares (C + 8 half steps), root and division; then three products
    fwd = C + 24
    R.close(y0, want['y'], mag['y'], fwd, 'y')
    if res:
        R.close(s0, want['r'], mag['r'], 1, 'r')
    else:
        assert s0 is x
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, r)]
    y, s = W.add_rms_norm(*leaves)
    assert torch.equal(y, y0)
    got = torch.autograd.grad((y, s) if res else y, [t for t in leaves if t is not None], (gy, gr) if res else gy)
    n = 1
    for v in rows:
        n *= v
    for name, g in zip(['g', 'gw'] + (['g'] if res else []), got):
        R.close(g, want[name], mag[name], 4 * fwd + (n if name == 'gw' else 0), name)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('C', [1, 7, 16, 100, 128, 130, 256, 512, 1000, 1024, 2048, 4100, 8192, 16400])
def test_norm_widths(dtype, C):
    for res in ('same', None, 'f32'):
        check_norm(dtype, (13,), C, res)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('rows', [(1,), (2, 3), (257,), (5, 411)], ids=str)
def test_norm_rows_and_strides(dtype, rows):
    for C in (48, 320):
        check_norm(dtype, rows, C, 'same', strided=True, seed=7)
        check_norm(dtype, rows, C, 'same', seed=8)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('C', [3, 16, 128, 1000, 2048, 4096, 9000])
@pytest.mark.parametrize('res', ['same', 'f32', None])
def test_norm_8bit(dtype, C, res):
    dt = DTYPES[dtype]
    x, w = (3 * rnd(1, 37, C)).to(dt), rnd(2, C)
    r = rnd(3, 37, C, dtype=torch.float32 if res == 'f32' else dt) if res else None
    x[5] = 0
    if r is not None:
        r[5] = 0
    q, scale, s = W.add_rms_norm_8bit(x, w, r)
    want, mag = (R.norm(x, w, r, mag=m) for m in (False, True))
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (37,)
    top = want['y'].abs().amax(-1)
    assert float(scale[5]) == 1.0 and not q[5].float().any()
    live = torch.arange(37, device='cuda') != 5
    slack = (C + 24) * R.U32 * mag['y'].amax(-1)
    assert ((scale.double() - top / 448).abs() <= 4 * R.U32 * top / 448 + slack / 448)[live].all()
    # half a step of e4m3 is 2^-4 of the value, 2^-10 near zero; the value before rounding carries the norm's fp32 error
    off = (q.double() * scale.double()[:, None] - want['y']).abs()
    tol = 2.0 ** -4 * want['y'].abs() + 2.0 ** -10 * scale.double()[:, None] + 2 * slack[:, None]
    assert (off <= tol).all(), float((off - tol).max())
    assert float(q.float().abs().amax(-1)[live].min()) == 448.0   # the largest value takes the largest code
    if res:
        R.close(s, want['r'], mag['r'], 1, 'r')


def test_norm_8bit_marks_a_row_that_is_not_finite():
    x, w = rnd(1, 4, 64), rnd(2, 64).abs() + 0.1
    x[1, 3] = float('nan')
    x[2, 5] = float('inf')
    q, scale, _ = W.add_rms_norm_8bit(x, w)
    assert torch.isnan(scale[1:3]).all() and torch.isnan(q[1].float()).all() and torch.isfinite(scale[[0, 3]]).all() and torch.isfinite(q[[0, 3]].float()).all()


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('C', [9, 61, 1021, 1999, 4095, 5001, 8191, 12001, 30001])
def test_norm_odd_widths(dtype, C):
    """rows that start at every offset of an access, contiguous and as slices of wider rows"""
    check_norm(dtype, (19,), C, 'same', seed=C)
    check_norm(dtype, (19,), C, 'f32' if C % 3 else 'same', strided=True, seed=C)
    x, w, r = rnd(1, 19, C, dtype=DTYPES[dtype]), rnd(2, C), rnd(3, 19, C, dtype=DTYPES[dtype])
    q, sc, _ = W.add_rms_norm_8bit(x, w, r)
    assert torch.equal(torch.isfinite(q.float()), torch.ones_like(q, dtype=torch.bool)) and float(q.float().abs().amax(-1).min()) == 448.0


@pytest.mark.parametrize('C', [5, 100, 1021, 3000, 8191, 16384, 16390])
def test_norm_backward_onto_the_gradient_it_adds(C):
    """the gradient of r may be where the sum goes, also with many rows a workgroup"""
    from wav2sleep_amd import lib
    rows = 2100
    r, w, g, gr = rnd(1, rows, C), rnd(2, C), rnd(3, rows, C), rnd(4, rows, C)
    rstd = torch.rsqrt(r.pow(2).mean(-1) + 1e-5)
    one, gw1, gw2 = torch.empty_like(r), torch.empty_like(w), torch.empty_like(w)
    lib.add_norm_bwd(r, w, rstd, g, gr, one, gw1, 1e-5)
    lib.add_norm_bwd(r, w, rstd, g, gr, gr, gw2, 1e-5)
    assert torch.equal(one, gr) and torch.equal(gw1, gw2)


def test_norm_8bit_of_the_smallest_numbers():
    """a row whose largest value over 448 is below every float: the codes stay numbers, and zeros zeros"""
    x = torch.tensor([[1.0, 0.0, -1.0, 0.5]], device='cuda').repeat(3, 4)
    w = torch.full((16,), 1e-43, device='cuda')
    q, scale, _ = W.add_rms_norm_8bit(x, w)
    v = q.float()
    assert (scale > 0).all() and torch.isfinite(v).all() and not v[x == 0].any()
    want = R.norm(x, w, None)['y']
    # rstd w and y are multiples of 2^-149, off by half of one each; the scale is exact; half a step of e4m3 is 2^-4 of y
    assert ((v.double() * scale.double()[:, None] - want).abs() <= 2.0 ** -4 * (want.abs() + 2.0 ** -149) + 2.0 ** -149).all()


def test_norm_of_more_rows_than_a_launch_takes():
    """narrow rows, sixteen a workgroup: 2^28 of them need more than 2^32 threads"""
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip('needs 8 GiB')
    rows = (1 << 28) + 5
    x = torch.empty(rows, 1, device='cuda', dtype=torch.bfloat16)
    x[:, 0] = (torch.arange(rows, device='cuda', dtype=torch.int32) % 7 - 3).to(torch.bfloat16)
    w = torch.full((1,), 2.0, device='cuda')
    y, _ = W.add_rms_norm(x, w, eps=0.0)
    assert torch.isnan(y[3]) and torch.equal(y[x != 0], (2 * torch.sign(x))[x != 0])   # x / |x| w, and a zero has no direction
    q, scale, _ = W.add_rms_norm_8bit(x, w)
    assert torch.equal(torch.sign(q.view(torch.int8).float()) < 0, x < 0) and (scale[x[:, 0] != 0] > 0).all()


# ------------------------------------------------------------------------------------------------------------------ edges that all share
def test_empty_calls():
    f = dict(device='cuda')
    w, b = rnd(1, 8, 4), rnd(2, 8)
    st = rnd(3, 2, 3, 8)
    y, last = W.short_conv(torch.empty(2, 0, 8, **f), w, b, state=st, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(last, st)
    assert W.short_conv(torch.empty(0, 5, 8, **f), w, b).shape == (0, 5, 8)
    A, h0 = -torch.rand(8, 4, **f), rnd(4, 2, 8, 4)
    e = torch.empty(2, 0, 8, **f)
    y, last = W.ssm_scan(e, e, A, torch.empty(2, 0, 4, **f), torch.empty(2, 0, 4, **f), state=h0, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(last, h0)
    y, last = W.ssm_scan(torch.empty(0, 3, 8, **f), torch.empty(0, 3, 8, **f), A, torch.empty(0, 3, 4, **f), torch.empty(0, 3, 4, **f), return_state=True)
    assert y.shape == (0, 3, 8) and last.shape == (0, 8, 4)
    y, r = W.add_rms_norm(torch.empty(0, 8, **f), b, torch.empty(0, 8, **f))
    assert y.shape == r.shape == (0, 8)
    # gradients of empty calls: the parameters' are zeros, a state's is what arrives at the final one
    for L, B in ((0, 2), (3, 0)):
        leaves = [t.requires_grad_(True) for t in (torch.empty(B, L, 8, **f), w.clone(), b.clone(), rnd(5, B, 3, 8))]
        y, last = W.short_conv(*leaves[:3], state=leaves[3], return_state=True)
        gs = rnd(6, *last.shape)
        gx, gw, gb, gst = torch.autograd.grad((y, last), leaves, (torch.empty_like(y), gs))
        assert not gw.any() and not gb.any() and torch.equal(gst, gs)
        h = rnd(7, B, 8, 4).requires_grad_(True)
        Ag = A.clone().requires_grad_(True)
        u = torch.empty(B, L, 8, **f).requires_grad_(True)
        bc = torch.empty(B, L, 4, **f)
        y, last = W.ssm_scan(u, u.detach(), Ag, bc, bc, state=h, return_state=True)
        gh = rnd(8, *last.shape)
        gu, gA, gst = torch.autograd.grad((y, last), [u, Ag, h], (torch.empty_like(y), gh))
        assert gu.shape == u.shape and not gA.any() and torch.equal(gst, gh)
    x, ww = torch.empty(0, 8, **f).requires_grad_(True), b.clone().requires_grad_(True)
    y, _ = W.add_rms_norm(x, ww)
    assert not torch.autograd.grad(y, ww, torch.empty_like(y))[0].any()


def test_partial_and_broadcast_gradients():
    """a gradient of the state alone, of y alone, an expanded one, and leaves that want none"""
    p = scan_inputs('f32', 2, 20, 16, 8, 1, seed=2)
    u, h = p['u'].clone().requires_grad_(True), p['state'].clone().requires_grad_(True)
    run = lambda: W.ssm_scan(u, p['dt'], p['A'], p['Bm'], p['Cm'], D=p['D'], z=p['z'], dt_bias=p['bias'], state=h, return_state=True)   # noqa: E731
    _, last = run()
    gu, gh = torch.autograd.grad(last, [u, h], p['gs'])
    args = (p['u'], p['dt'], p['A'], p['Bm'], p['Cm'], p['D'], p['z'], p['bias'])
    want, mag = (R.scan(*args, state=p['state'], gs=p['gs'], mag=m) for m in (False, True))
    R.close(gu, want['gu'], mag['gu'], 110 * 44, 'gu')
    R.close(gh, want['gstate'], mag['gstate'], 110 * 44, 'gstate')
    y, _ = run()
    gu, = torch.autograd.grad(y.sum(), [u])   # an expanded gradient
    want, mag = (R.scan(*args, state=p['state'], gy=torch.ones_like(p['u']), mag=m) for m in (False, True))
    R.close(gu, want['gu'], mag['gu'], 110 * 44, 'gu of a sum')
    x, w = rnd(1, 2, 9, 16).requires_grad_(True), rnd(2, 16, 4)
    y, last = W.short_conv(x, w, None, None, return_state=True)
    gx, = torch.autograd.grad(last, x, torch.ones_like(last), retain_graph=True)
    assert torch.equal(gx[:, -3:], torch.ones_like(gx[:, -3:])) and not gx[:, :-3].any()
    gx, = torch.autograd.grad(y.sum(), x)
    want, mag = (R.conv(x, w, None, False, gy=torch.ones_like(x), mag=m) for m in (False, True))
    R.close(gx, want['gx'], mag['gx'], 16, 'gx of a sum')


def test_channel_strides_are_copied():
    p = scan_inputs('f32', 2, 12, 16, 8, 1, seed=6)
    t = {k: p[k].transpose(-1, -2).contiguous().transpose(-1, -2) for k in ('u', 'dt', 'Bm', 'Cm', 'z')}
    a = W.ssm_scan(p['u'], p['dt'], p['A'], p['Bm'], p['Cm'], z=p['z'])
    assert torch.equal(a, W.ssm_scan(t['u'], t['dt'], p['A'].t().contiguous().t(), t['Bm'], t['Cm'], z=t['z']))
    w = rnd(1, 16, 4)
    assert torch.equal(W.short_conv(p['u'], w), W.short_conv(t['u'], w.t().contiguous().t()))
    assert torch.equal(W.add_rms_norm(p['u'], w[:, 0].contiguous(), p['z'])[0], W.add_rms_norm(t['u'], w[:, 0], t['z'])[0])


def test_offsets_beyond_32_bits():
    """sequences that lie more than 2^31 elements into their tensors give what they give alone"""
    B, L, D, N = 2, 33, 16, 16
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 40 GiB')
    far = (1 << 31) + 4096
    big = torch.empty(far + B * L * D, device='cuda', dtype=torch.bfloat16)
    p = scan_inputs('bf16', B, L, D, N, 1, seed=12)
    for k in ('u', 'dt', 'z'):
        v = torch.as_strided(big, (B, L, D), (far, D, 1))
        v.copy_(p[k])
        y = W.short_conv(v, rnd(1, D, 4))
        assert torch.equal(y, W.short_conv(p[k], rnd(1, D, 4)))
        if k == 'u':
            y = W.ssm_scan(v, p['dt'], p['A'], p['Bm'], p['Cm'], z=p['z'])
            assert torch.equal(y, W.ssm_scan(p['u'], p['dt'], p['A'], p['Bm'], p['Cm'], z=p['z']))
            r = W.add_rms_norm(v, rnd(2, D), v)[0]
            assert torch.equal(r, W.add_rms_norm(p['u'], rnd(2, D), p['u'])[0])


# ------------------------------------------------------------------------------------------------------------------ together, streams, graphs
class Block:
    """one mixer block in plain calls: norm, projection, short convolution, projection, scan, projection"""

    def __init__(self, F=32, E=48, N=8, rank=4, K=4, dtype=torch.float32, seed=100):
        s = iter(range(seed, seed + 20))
        self.E, self.N, self.rank, self.K = E, N, rank, K
        self.w = 1 + 0.1 * rnd(next(s), F)
        self.inp = (rnd(next(s), 2 * E, F) / F ** 0.5).to(dtype)
        self.cw, self.cb = rnd(next(s), E, K) / 2, 0.1 * rnd(next(s), E)
        self.xp = (rnd(next(s), rank + 2 * N, E) / E ** 0.5).to(dtype)
        self.dtp = (rnd(next(s), E, rank) / rank ** 0.5).to(dtype)
        self.bias = -3 + 0.3 * rnd(next(s), E)
        self.A = -(0.2 + torch.rand(E, N, device='cuda') * 4)
        self.D = rnd(next(s), E)
        self.out = (rnd(next(s), F, E) / E ** 0.5).to(dtype)

    def parts(self, uz, dbc):
        E, N, r = self.E, self.N, self.rank
        return dbc[..., :r], dbc[..., r:r + N], dbc[..., r + N:], uz[..., :E], uz[..., E:]

    def prompt(self, x, res, lengths=None, conv_state=None, state=None):
        y, r = W.add_rms_norm(x, self.w, res)
        uz = y @ self.inp.t()
        u, cs = W.short_conv(uz[..., :self.E], self.cw, self.cb, state=conv_state, lengths=lengths, return_state=True)
        dbc = u @ self.xp.t()
        low, B, C, _, z = self.parts(uz, dbc)
        s, h = W.ssm_scan(u, low @ self.dtp.t(), self.A, B, C, D=self.D, z=z, dt_bias=self.bias, state=state, lengths=lengths, return_state=True)
        return s @ self.out.t(), r, cs, h

    def step(self, x, res, cs, h):
        y, r = W.add_rms_norm(x, self.w, res)
        uz = y @ self.inp.t()
        u = W.short_conv_step(uz[..., :self.E], cs, self.cw, self.cb)
        dbc = u @ self.xp.t()
        low, B, C, _, z = self.parts(uz, dbc)
        return W.ssm_step(u, low @ self.dtp.t(), self.A, B, C, h, D=self.D, z=z, dt_bias=self.bias) @ self.out.t(), r

    def reference(self, x, res):
        d = R.d64
        n = R.norm(x, self.w, res)
        uz = n['y'] @ d(self.inp).t()
        u = R.conv(uz[..., :self.E], self.cw, self.cb)['y']
        dbc = u @ d(self.xp).t()
        low, B, C, _, z = self.parts(uz, dbc)
        s = R.scan(u, low @ d(self.dtp).t(), self.A, B[:, :, None], C[:, :, None], self.D, z, self.bias)['y']
        return s @ d(self.out).t(), n['r']


def test_a_prompt_then_single_positions():
    blk, B, L = Block(), 3, 40
    x, res = rnd(1, B, L, 32), rnd(2, B, L, 32)
    want, _ = blk.reference(x, res)
    size = float(want.abs().max())
    n = torch.tensor([17, 1, 9], device='cuda', dtype=torch.int32)   # prompts of unequal length, then one position at a time
    out, _, cs, h = blk.prompt(x, res, lengths=n)
    for b in range(B):
        k = int(n[b])
        # three matrix products of up to 48 terms and two operators of ~100 half steps on values that the chain may enlarge tenfold: 1e-5 of the largest is 160 half steps
        assert float((out[b, :k].double() - want[b, :k]).abs().max()) <= 1e-4 * size
    for i in range(20):
        at = n.long() + i
        ar = torch.arange(B, device='cuda')
        y, _ = blk.step(x[ar, at], res[ar, at], cs, h)
        assert float((y.double() - want[ar, at]).abs().max()) <= 1e-4 * size, i


def test_block_gradients_of_the_whole_run():
    blk, B, L = Block(), 2, 25
    x, res, g = rnd(1, B, L, 32), rnd(2, B, L, 32), rnd(3, B, L, 32)
    x.requires_grad_(True)
    blk.A.requires_grad_(True)
    blk.cw.requires_grad_(True)
    out = blk.prompt(x, res)[0]
    got = torch.autograd.grad((out * g).sum(), [x, blk.A, blk.cw])
    for t, gk, seed in zip((x, blk.A, blk.cw), got, (4, 5, 6)):
        way, eps, keep = rnd(seed, *t.shape).double(), 1e-6, t
        vals = []
        for s in (1, -1):
            moved = (t.detach().double() + s * eps * way)
            if t is x:
                vals.append(float((blk.reference(moved, res)[0] * g.double()).sum()))
            else:
                name = 'A' if t is blk.A else 'cw'
                setattr(blk, name, moved)
                vals.append(float((blk.reference(x, res)[0] * g.double()).sum()))
                setattr(blk, name, keep)
        want, have = (vals[0] - vals[1]) / (2 * eps), float((gk.double() * way).sum())
        assert abs(have - want) <= 1e-4 * float((gk.double() * way).abs().sum()), (have, want)


def test_side_stream_and_two_calls_at_once():
    p, q = scan_inputs('bf16', 4, 200, 64, 16, 1, seed=1), scan_inputs('bf16', 4, 200, 64, 16, 1, seed=50)
    call = lambda v: W.ssm_scan(v['u'], v['dt'], v['A'], v['Bm'], v['Cm'], D=v['D'], z=v['z'], dt_bias=v['bias'])   # noqa: E731
    a, b = call(p), call(q)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            a1 = call(p)
        with torch.cuda.stream(s2):
            b1 = call(q)
        torch.cuda.synchronize()
        assert torch.equal(a, a1) and torch.equal(b, b1)


def test_steps_in_inference_mode():
    p = scan_inputs('bf16', 3, 4, 16, 16, 1, seed=20)
    w = rnd(1, 16, 4)
    calls = lambda: (W.short_conv_step(p['u'][:, 0], torch.zeros(3, 3, 16, device='cuda', dtype=torch.bfloat16), w),   # noqa: E731
                     W.ssm_step(p['u'][:, 0], p['dt'][:, 0], p['A'], p['Bm'][:, 0], p['Cm'][:, 0], torch.zeros(3, 16, 16, device='cuda')),
                     W.ssm_scan(p['u'], p['dt'], p['A'], p['Bm'], p['Cm']), W.short_conv(p['u'], w), W.add_rms_norm(p['u'], w[:, 0], p['z'])[1])
    want = calls()
    with torch.inference_mode():
        got = calls()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals_of_sizes():
    f = dict(device='cuda')
    big = torch.zeros(1, 1, 8, **f).expand(1, (1 << 30) + 1, 8)   # (no memory behind it)
    w = rnd(1, 8, 4)
    with pytest.raises(ValueError):
        W.short_conv(big, w)
    bc = torch.zeros(1, 1, 4, **f).expand(1, (1 << 30) + 1, 4)
    with pytest.raises(ValueError):
        W.ssm_scan(big, big, -w, bc, bc)
    rows = torch.zeros(1, 8, **f).expand(1 << 31, 8)
    for op in (W.add_rms_norm, W.add_rms_norm_8bit):
        with pytest.raises(ValueError):
            op(rows, w[:, 0].contiguous())


def test_graphs_replay_forward_and_steps():
    blk, B = Block(), 4
    x, res = rnd(1, B, 64, 32), rnd(2, B, 64, 32)
    big = scan_inputs('f32', 1, 2000, 16, 16, 1, seed=9)   # (a call that needs scratch memory)
    scan = lambda: W.ssm_scan(big['u'], big['dt'], big['A'], big['Bm'], big['Cm'], D=big['D'], z=big['z'], dt_bias=big['bias'])   # noqa: E731

    def work():
        out, _, cs, h = blk.prompt(x, res)
        y, _ = blk.step(x[:, 0], res[:, 0], cs, h)
        return out, y, cs, h, scan()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work())
        graphs.append(g)
    for k in range(3):
        x.copy_(rnd(60 + k, B, 64, 32))
        big['u'].copy_(rnd(70 + k, 1, 2000, 16))
        want = work()
        torch.cuda.synchronize()
        for g, o in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(o, want):
                assert torch.equal(a, b)


def test_graph_replays_a_backward():
    p = scan_inputs('f32', 2, 300, 32, 16, 1, seed=14)
    x, w, b = rnd(1, 2, 300, 32), rnd(2, 32, 4), rnd(3, 32)
    nw = rnd(4, 32)

    def work():
        xs, ws, bs, u0, A, nws = (t.detach().requires_grad_(True) for t in (x, w, b, p['u'], p['A'], nw))
        y, r = W.add_rms_norm(xs, nws, u0)
        c = W.short_conv(y, ws, bs)
        o = W.ssm_scan(c, p['dt'], A, p['Bm'], p['Cm'], z=r)
        return torch.autograd.grad(o, [xs, ws, bs, u0, A, nws], p['gy'])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    for k in range(3):
        x.copy_(rnd(80 + k, 2, 300, 32))
        want = work()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    E = W.lib.W2SError
    p = scan_inputs('f32', 2, 6, 8, 4, 2, seed=1)
    good = dict(u=p['u'], dt=p['dt'], A=p['A'], B=p['Bm'], C=p['Cm'], D=p['D'], z=p['z'], dt_bias=p['bias'], state=p['state'])
    W.ssm_scan(**good)
    bad = [(dict(u=p['u'].double()), ValueError), (dict(dt=p['dt'].bfloat16()), ValueError), (dict(A=p['A'].bfloat16()), ValueError), (dict(A=p['A'][:4]), ValueError),
           (dict(A=rnd(1, 8, 65)), ValueError), (dict(B=p['Bm'][:, :, :, :3]), ValueError), (dict(B=rnd(1, 2, 6, 3, 4)), ValueError), (dict(C=p['Cm'][:, :, :1]), ValueError),
           (dict(z=p['z'][:1]), ValueError), (dict(state=p['state'].bfloat16()), ValueError), (dict(D=p['D'][:3]), ValueError), (dict(dt=None), TypeError),
           (dict(lengths=torch.tensor([1, 2], device='cuda')), ValueError), (dict(lengths=torch.tensor([1], device='cuda', dtype=torch.int32)), ValueError),
           (dict(dt=p['dt'].cpu()), E), (dict(lengths=torch.tensor([1, 2], dtype=torch.int32)), E), (dict(u=p['u'][0]), ValueError), (dict(B=None), TypeError)]
    for kw, err in bad:
        with pytest.raises(err):
            W.ssm_scan(**{**good, **kw})
    row = {k: (v[:, 0] if k in ('u', 'dt', 'B', 'C', 'z') else v) for k, v in good.items()}
    W.ssm_step(**row)
    with pytest.raises(TypeError):
        W.ssm_step(**{**row, 'state': None})
    with pytest.raises(ValueError):   # neither the same tensor nor apart from it
        big = torch.zeros(2 * 8 * 4 + 4, device='cuda')
        W.ssm_step(**{**row, 'state': big[:64].view(2, 8, 4)}, state_out=big[4:].view(2, 8, 4))
    with pytest.raises(ValueError):
        W.ssm_step(**{**row, 'state': rnd(1, 2, 4, 8).transpose(1, 2)})
    with pytest.raises(E):
        W.ssm_step(**{**row, 'u': row['u'].clone().requires_grad_(True)})
    with pytest.raises(E):
        W.ssm_step(**row, state_out=torch.zeros_like(p['state']).requires_grad_(True))
    x, w = rnd(1, 2, 6, 8), rnd(2, 8, 4)
    for args, kw, err in [((x, rnd(1, 8, 9)), {}, ValueError), ((x, rnd(1, 7, 4)), {}, ValueError), ((x, w.bfloat16()), {}, ValueError), ((x, w, w[:, 0], 'relu'), {}, ValueError),
                          ((x[0], w), {}, ValueError), ((x, w), dict(state=rnd(1, 2, 4, 8)), ValueError), ((x, w), dict(state=rnd(1, 2, 3, 8).bfloat16()), ValueError),
                          ((x.half(), w, w[:, 0].half()), {}, ValueError), ((x, w), dict(lengths=torch.ones(2, device='cuda')), ValueError), ((x, w.cpu()), {}, E)]:
        with pytest.raises(err):
            W.short_conv(*args, **kw)
    with pytest.raises(E):
        W.short_conv_step(x[:, 0].clone().requires_grad_(True), rnd(1, 2, 3, 8), w)
    with pytest.raises(ValueError):
        W.short_conv_step(x[:, 0], rnd(1, 2, 2, 8), w)
    for args, err in [((x, w[:, 0].bfloat16()), ValueError), ((x, rnd(1, 7)), ValueError), ((x, rnd(1, 8), x.bfloat16()), ValueError), ((x, rnd(1, 8), x[:1]), ValueError),
                      ((x.bfloat16(), rnd(1, 8), x.half()), ValueError), ((x, None), TypeError), ((x, rnd(1, 8), None, -1.0), ValueError), ((x, rnd(1, 8), None, float('nan')), ValueError)]:
        for f in (W.add_rms_norm, W.add_rms_norm_8bit):
            with pytest.raises(err):
                f(*args)
    with pytest.raises(E):
        W.add_rms_norm_8bit(x.clone().requires_grad_(True), rnd(1, 8))
    far = torch.zeros(5 * (1 << 22) + 64, device='cuda').as_strided((2, 6, 8), (8, 1 << 22, 1))   # positions further apart than the offsets inside a tile reach
    with pytest.raises(E):
        W.ssm_scan(**{**good, 'u': far})
    u = p['u'].clone().requires_grad_(True)   # first order only
    y = W.ssm_scan(**{**good, 'u': u})
    g, = torch.autograd.grad(y.sum(), u, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
