"""Measured cases of the state space mixer's operators: the short causal convolution, the selective scan and the root-mean-square norm with
the residual's addition, over whole recordings, in training and for single epochs of a stream.

`own = False` computes the operators from elementary torch operations in 32 bits; `own = True` calls wav2sleep_amd's kernels.
Shapes: B sequences of L positions (epochs of 30 s, or finer), D channels, N states per channel, G groups of channels that share B and C.
"""
import math

import torch

own = False

_TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
_FP8_MAX = 448.0   # largest finite e4m3 value
_EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a batch of sixteen 8-hour recordings, 960 epochs, twice the model's 128 features; the states go on to the next call
        dict(name='conv_night', op='conv', dtype='f32', B=16, L=960, D=256, K=4, ragged=False, carry=True),
        # a training pass over recordings of unequal length in 16 bits, an odd maximum length
        dict(name='conv_train_ragged', op='conv_train', dtype='bf16', B=8, L=2047, D=1536, K=4, ragged=True, carry=False),
        # the newest epoch of 24 live recordings: the smallest call
        dict(name='conv_stream', op='conv_step', dtype='f32', B=24, D=256, K=4),
        # the scan over the same sixteen nights, gated, from a given state
        dict(name='scan_night', op='scan', dtype='f32', B=16, L=960, D=256, N=16, G=1, gate=True, ragged=False, carry=True),
        # ONE long recording at a fine resolution: few rows, a long axis
        dict(name='scan_long_row', op='scan', dtype='bf16', B=1, L=16384, D=512, N=16, G=1, gate=True, ragged=False, carry=False),
        # a training pass over sixteen nights
        dict(name='scan_train', op='scan_train', dtype='f32', B=16, L=960, D=256, N=16, G=1, gate=True, ragged=False, carry=False),
        # a wide mixer in 16 bits, three groups, recordings of unequal length
        dict(name='scan_train_ragged', op='scan_train', dtype='bf16', B=4, L=2047, D=1536, N=16, G=3, gate=True, ragged=True, carry=False),
        # the newest epoch of 256 live recordings
        dict(name='scan_stream', op='scan_step', dtype='f32', B=256, D=512, N=16, G=1, gate=True),
        # the token rows of sixteen nights (16 x 960 epochs x 5 tokens), 128 features
        dict(name='norm_tokens', op='norm', dtype='f32', rows=76800, C=128),
        # a training pass over wide rows in 16 bits, an odd number of them
        dict(name='norm_train', op='norm_train', dtype='bf16', rows=16383, C=2048),
        # rows for an 8-bit matrix product
        dict(name='norm_8bit', op='norm_8bit', dtype='bf16', rows=16384, C=4096),
        # a handful of rows of an odd width
        dict(name='norm_8bit_few', op='norm_8bit', dtype='f16', rows=5, C=1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['conv', 'conv_train', 'conv_step', 'scan', 'scan', 'scan_train', 'scan_train', 'scan_step', 'norm', 'norm_train', 'norm_8bit'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    yes = lambda: rng.random() < 0.5   # noqa: E731
    if op in ('norm', 'norm_train', 'norm_8bit'):
        C = _log(rng, 16, 8192)
        return dict(op=op, dtype=dtype, rows=min(_log(rng, 1, 131072), 33_000_000 // C), C=C)
    if op == 'conv_step':
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 512), D=_log(rng, 16, 4096), K=rng.randint(2, 6))
    G = rng.choice([1, 1, 1, 2, 4])
    D = G * max(1, _log(rng, 16, 4096) // G)
    N = rng.choice([8, 16, 16, 16, 24, 32, 64])
    if op == 'scan_step':
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 512), D=D, N=N, G=G, gate=yes())
    L = _log(rng, 1, 16384)
    if op in ('conv', 'conv_train'):
        return dict(op=op, dtype=dtype, B=max(1, min(_log(rng, 1, 64), 25_000_000 // (L * D))), L=L, D=D, K=rng.randint(2, 6), ragged=yes(), carry=yes())
    D = max(G, min(D, 190_000_000 // (L * N) // G * G))
    return dict(op=op, dtype=dtype, B=max(1, min(_log(rng, 1, 64), 190_000_000 // (L * D * N))), L=L, D=D, N=N, G=G, gate=yes(), ragged=yes(), carry=yes())


def work(case):
    s, op = _BYTES[case['dtype']], case['op']
    if op in ('norm', 'norm_train', 'norm_8bit'):
        R, C = case['rows'], case['C']
        if op == 'norm':        # x, residual in; sum, normalised out
            return dict(bytes=4 * s * R * C + 4 * C, flops=5 * R * C)
        if op == 'norm_8bit':   # x, residual in; sum, one byte and a scale a row out
            return dict(bytes=(3 * s + 1) * R * C + 4 * R + 4 * C, flops=8 * R * C)
        # x, residual, two gradients in; sum, normalised, the gradient that both addends share out
        return dict(bytes=7 * s * R * C + 8 * C, flops=14 * R * C)
    B, D = case['B'], case['D']
    if op == 'conv_step':
        return dict(bytes=2 * s * B * D * case['K'] + 4 * D * (case['K'] + 1), flops=2 * B * D * case['K'])
    if op == 'scan_step':
        N, G = case['N'], case['G']
        return dict(bytes=8 * B * D * N + (4 if case['gate'] else 3) * s * B * D + 2 * s * B * G * N + 4 * D * (N + 2), flops=7 * B * D * N)
    E = B * case['L'] * D
    if op in ('conv', 'conv_train'):
        K = case['K']
        edge = 2 * s * B * (K - 1) * D if case['carry'] else 0
        if op == 'conv':        # x in, y out
            return dict(bytes=2 * s * E + 4 * D * (K + 1) + edge, flops=2 * K * E)
        return dict(bytes=4 * s * E + 8 * D * (K + 1) + 2 * edge, flops=8 * K * E)   # x, gy in; y, gx out
    N, G = case['N'], case['G']
    bc = 2 * s * B * case['L'] * G * N
    edge = 8 * B * D * N if case['carry'] else 0
    if op == 'scan':            # u, dt, (z) in; y out
        return dict(bytes=(4 if case['gate'] else 3) * s * E + bc + 4 * D * (N + 2) + edge, flops=7 * E * N)
    # u, dt, (z), gy in; y and the gradients of u, dt, (z) out
    return dict(bytes=(8 if case['gate'] else 6) * s * E + 2 * bc + 8 * D * (N + 2) + 2 * edge, flops=25 * E * N)


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    f32, io = torch.float32, _TYPES[case['dtype']]
    normal = lambda *shape: torch.randn(*shape, device='cuda', dtype=f32, generator=g)   # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, device='cuda', dtype=f32, generator=g)   # noqa: E731
    st = dict(case)
    op = case['op']
    if op in ('norm', 'norm_train', 'norm_8bit'):
        R, C = case['rows'], case['C']
        st['x'], st['res'] = normal(R, C).to(io), (2.0 * normal(R, C)).to(io)
        st['w'] = 1.0 + 0.2 * normal(C)
        if op == 'norm_train':
            st['gy'], st['gr'] = normal(R, C).to(io), normal(R, C).to(io)
            for k in ('x', 'res', 'w'):
                st[k].requires_grad_(True)
        return st
    B, D = case['B'], case['D']
    if op in ('conv', 'conv_train', 'conv_step'):
        K = case['K']
        st['w'], st['b'] = normal(D, K) / math.sqrt(K), 0.1 * normal(D)
        if op == 'conv_step':
            st['x'], st['state'] = normal(B, D).to(io), normal(B, K - 1, D).to(io)
            st['out'] = torch.empty_like(st['state'])
            return st
        wide = normal(B, case['L'], 2 * D).to(io)   # the projection that holds both the convolution's input and the gate
        st['x'] = wide[..., :D].detach()
        st['state'] = normal(B, K - 1, D).to(io) if case['carry'] else None
        if op == 'conv_train':
            st['gy'] = normal(B, case['L'], D).to(io)
            st['gs'] = normal(B, K - 1, D).to(io) if case['carry'] else None
    else:
        N, G = case['N'], case['G']
        step = op == 'scan_step'
        rows = (B,) if step else (B, case['L'])
        u = normal(*rows, D)
        st['u'] = (u * torch.sigmoid(u)).to(io)
        st['dt'] = (0.5 * normal(*rows, D)).to(io)
        first = torch.exp(uniform(D) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))   # time steps from 0.001 to 0.1
        st['bias'] = first + torch.log(-torch.expm1(-first))
        st['A'] = -torch.arange(1, N + 1, device='cuda', dtype=f32)[None, :] * torch.exp(0.2 * normal(D, N))
        st['Dp'] = 1.0 + 0.1 * normal(D)
        bc = normal(*rows, 2 * G * N).to(io)        # the projection that holds B and C
        st['Bm'], st['Cm'] = (bc[..., q * G * N:(q + 1) * G * N].unflatten(-1, (G, N)).detach() for q in (0, 1))
        wide = normal(*rows, 2 * D).to(io)
        st['z'] = wide[..., D:].detach() if case['gate'] else None
        if step:
            st['state'] = normal(B, D, N)
            st['out'] = torch.empty_like(st['state'])
            return st
        st['state'] = normal(B, D, N) if case['carry'] else None
        if op == 'scan_train':
            st['gy'] = normal(B, case['L'], D).to(io)
            st['gs'] = normal(B, D, N) if case['carry'] else None
    if case['ragged']:
        n = (uniform(B) * (case['L'] + 1)).to(torch.int32)
        n[0] = case['L']
        st['lengths'] = n.clamp_(max=case['L'])
    else:
        st['lengths'] = None
    if op.endswith('train'):
        for k in ('x', 'w', 'b', 'u', 'dt', 'A', 'Bm', 'Cm', 'Dp', 'z', 'bias', 'state'):
            if st.get(k) is not None:
                st[k].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------------------------------------------- plain forms (32 bits)
def _silu_pair(x):
    s = torch.sigmoid(x)
    return x * s, s * (1.0 + x * (1.0 - s))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-torch.abs(x)))


def _alive(st):
    """[B, L, 1] truth values: positions inside their sequence"""
    n = st['lengths']
    L = st['L']
    if n is None:
        return torch.ones(st['B'], L, 1, device='cuda', dtype=torch.bool)
    return (torch.arange(L, device='cuda')[None, :] < n[:, None].long())[..., None]


def _plain_conv(st, train):
    K, L = st['K'], st['L']
    alive = _alive(st)
    x = torch.where(alive, st['x'].detach().float(), 0.0)
    w, b = st['w'].detach(), st['b'].detach()
    first = st['state'].detach().float() if st['state'] is not None else x.new_zeros(st['B'], K - 1, st['D'])
    full = torch.cat([first, x], dim=1)
    win = full.unfold(1, K, 1)                                       # [B, L, D, K]
    z = (win * w).sum(-1) + b
    act, slope = _silu_pair(z)
    y = torch.where(alive, act, 0.0).to(st['x'].dtype)
    n = st['lengths'].long() if st['lengths'] is not None else torch.full((st['B'],), L, device='cuda')
    at = (n[:, None] + torch.arange(K - 1, device='cuda'))[..., None].expand(-1, -1, st['D'])   # rows n .. n + K - 2 of `full`
    last = torch.gather(full, 1, at).to(st['x'].dtype)
    if not train:
        return [y, last] if st['carry'] else [y]
    gz = torch.where(alive, st['gy'].float() * slope, 0.0)
    gw = torch.stack([(gz * win[..., k]).sum((0, 1)) for k in range(K)], dim=1)
    gfull = torch.zeros_like(full)
    for k in range(K):
        gfull[:, k:k + L] += gz * w[:, k]
    if st['carry']:
        gfull.scatter_add_(1, at, st['gs'].float())
    gx = torch.where(alive, gfull[:, K - 1:], 0.0).to(st['x'].dtype)
    out = [y, gx, gw, gz.sum((0, 1))]
    return out + [last, gfull[:, :K - 1].to(st['x'].dtype)] if st['carry'] else out


def _recur(a, x):
    """h_t = a_t h_{t-1} + x_t along dimension 1 from zero, by doubling"""
    n, span = a.shape[1], 1
    while span < n:
        x = torch.cat([x[:, :span], x[:, span:] + a[:, span:] * x[:, :-span]], dim=1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], dim=1)
        span *= 2
    return x


def _per_channel(m, D):
    """[B, L, G, N] of a group -> [B, L, D, N] of its channels"""
    return m.repeat_interleave(D // m.shape[2], dim=2)


def _plain_scan(st, train):
    D, G = st['D'], st['G']
    alive = _alive(st)
    clean = lambda t: torch.where(alive, t.detach().float(), 0.0)   # noqa: E731
    u, A, Dp = clean(st['u']), st['A'].detach(), st['Dp'].detach()
    raw = clean(st['dt']) + st['bias'].detach()
    delta = torch.where(alive, _softplus(raw), 0.0)
    alive4 = alive[..., None]
    Bm = _per_channel(torch.where(alive4, st['Bm'].detach().float(), 0.0), D)
    Cm = _per_channel(torch.where(alive4, st['Cm'].detach().float(), 0.0), D)
    a = torch.exp(delta[..., None] * A)
    x = (delta * u)[..., None] * Bm
    h0 = st['state'].detach() if st['state'] is not None else torch.zeros(st['B'], D, st['N'], device='cuda')
    if st['carry']:
        x[:, 0] += a[:, 0] * h0
    h = _recur(a, x)
    del x
    pre = (h * Cm).sum(-1) + Dp * u
    if st['gate']:
        gate, slope = _silu_pair(clean(st['z']))
    y = (pre * gate if st['gate'] else pre).to(st['u'].dtype)
    last = h[:, -1].clone() if st['carry'] else None
    if not train:
        return [y, last] if st['carry'] else [y]
    gy = clean(st['gy'])
    gp = gy * gate if st['gate'] else gy
    gh = gp[..., None] * Cm
    if st['carry']:
        gh[:, -1] += st['gs']
    ahead = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], dim=1)
    gh = _recur(ahead.flip(1), gh.flip(1)).flip(1)
    del ahead
    group = lambda t: t.unflatten(2, (G, D // G)).sum(3)   # noqa: E731
    io = st['u'].dtype
    gC = group(gp[..., None] * h).to(io)
    gB = group(gh * (delta * u)[..., None]).to(io)
    sB = (gh * Bm).sum(-1)
    back = torch.cat([h0[:, None], h[:, :-1]], dim=1) * a * gh
    del Bm, Cm, h
    gA = (back * delta[..., None]).sum((0, 1))
    gdelta = (back * A).sum(-1) + u * sB
    graw = torch.where(alive, gdelta * torch.sigmoid(raw), 0.0)
    out = [y, (delta * sB + Dp * gp).to(io), graw.to(io), gA, gB, gC, (gp * u).sum((0, 1)), graw.sum((0, 1))]
    if st['gate']:
        out.append((gy * pre * slope).to(io))
    return out + [last, a[:, 0] * gh[:, 0]] if st['carry'] else out


def _plain_conv_step(st):
    full = torch.cat([st['state'].float(), st['x'].float()[:, None]], dim=1)
    z = (full * st['w'].t()).sum(1) + st['b']
    return [(z * torch.sigmoid(z)).to(st['x'].dtype), full[:, 1:].to(st['x'].dtype)]


def _plain_scan_step(st):
    D = st['D']
    u = st['u'].float()
    delta = _softplus(st['dt'].float() + st['bias'])
    Bm, Cm = (st[k].float().repeat_interleave(D // st['G'], dim=1) for k in ('Bm', 'Cm'))
    h = torch.exp(delta[..., None] * st['A']) * st['state'] + (delta * u)[..., None] * Bm
    y = (h * Cm).sum(-1) + st['Dp'] * u
    if st['gate']:
        y = y * _silu_pair(st['z'].float())[0]
    return [y.to(st['u'].dtype), h]


def _plain_norm(st):
    io, w = st['x'].dtype, st['w'].detach()
    r = st['x'].detach().float() + st['res'].detach().float()
    rstd = torch.rsqrt((r * r).mean(-1, keepdim=True) + _EPS)
    n = r * rstd
    if st['op'] == 'norm':
        return [(n * w).to(io), r.to(io)]
    if st['op'] == 'norm_8bit':
        y = n * w
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top > 0.0, top / _FP8_MAX, 1.0)
        return [torch.clamp(y / scale, -_FP8_MAX, _FP8_MAX).to(torch.float8_e4m3fn), scale[:, 0], r.to(io)]
    gy = st['gy'].float()
    gn = gy * w
    gx = (rstd * (gn - n * (gn * n).mean(-1, keepdim=True)) + st['gr'].float()).to(io)
    return [(n * w).to(io), r.to(io), gx, gx, (gy * n).sum(0)]


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    st, op = state, state['op']
    if not own:
        if op in ('conv', 'conv_train'):
            return _plain_conv(st, op == 'conv_train')
        if op in ('scan', 'scan_train'):
            return _plain_scan(st, op == 'scan_train')
        return {'conv_step': _plain_conv_step, 'scan_step': _plain_scan_step}.get(op, _plain_norm)(st)
    import wav2sleep_amd as W
    if op in ('conv', 'conv_train'):
        y = W.short_conv(st['x'], st['w'], st['b'], activation='silu', state=st['state'], lengths=st['lengths'], return_state=st['carry'])
        if op == 'conv':
            return list(y) if st['carry'] else [y]
        if not st['carry']:
            return [y, *torch.autograd.grad(y, (st['x'], st['w'], st['b']), st['gy'])]
        y, last = y
        gx, gw, gb, gs = torch.autograd.grad((y, last), (st['x'], st['w'], st['b'], st['state']), (st['gy'], st['gs']))
        return [y, gx, gw, gb, last, gs]
    if op in ('scan', 'scan_train'):
        y = W.ssm_scan(st['u'], st['dt'], st['A'], st['Bm'], st['Cm'], D=st['Dp'], z=st['z'], dt_bias=st['bias'], dt_softplus=True,
                       state=st['state'], lengths=st['lengths'], return_state=st['carry'])
        if op == 'scan':
            return list(y) if st['carry'] else [y]
        leaves = [st[k] for k in ('u', 'dt', 'A', 'Bm', 'Cm', 'Dp', 'bias')] + ([st['z']] if st['gate'] else [])
        if not st['carry']:
            return [y, *torch.autograd.grad(y, leaves, st['gy'])]
        y, last = y
        *grads, gs = torch.autograd.grad((y, last), leaves + [st['state']], (st['gy'], st['gs']))
        return [y, *grads, last, gs]
    if op == 'conv_step':
        return [W.short_conv_step(st['x'], st['state'], st['w'], st['b'], activation='silu', state_out=st['out']), st['out']]
    if op == 'scan_step':
        return [W.ssm_step(st['u'], st['dt'], st['A'], st['Bm'], st['Cm'], st['state'], D=st['Dp'], z=st['z'], dt_bias=st['bias'],
                           dt_softplus=True, state_out=st['out']), st['out']]
    if op == 'norm_8bit':
        return list(W.add_rms_norm_8bit(st['x'], st['w'], residual=st['res'], eps=_EPS))
    y, r = W.add_rms_norm(st['x'], st['w'], residual=st['res'], eps=_EPS)
    if op == 'norm':
        return [y, r]
    return [y, r, *torch.autograd.grad((y, r), (st['x'], st['res'], st['w']), (st['gy'], st['gr']))]


# ---------------------------------------------------------------------------------------------------------------- 64 bits, position by position
def exact(case, seed):
    st = prepare(case, seed)
    op = case['op']
    d = {k: (v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in st.items()}
    train = op.endswith('train')
    if train:
        d = {k: (v.requires_grad_(True) if isinstance(st[k], torch.Tensor) and st[k].requires_grad else v) for k, v in d.items()}
    F = torch.nn.functional
    if op in ('norm', 'norm_train', 'norm_8bit'):
        r = d['x'] + d['res']
        y = r / torch.sqrt(r.pow(2).sum(-1, keepdim=True) / case['C'] + _EPS) * d['w']
        if op == 'norm':
            return [y, r]
        if op == 'norm_train':
            return [y.detach(), r.detach(), *torch.autograd.grad((y, r), (d['x'], d['res'], d['w']), (d['gy'], d['gr']))]
        scale = y.abs().max(-1).values / _FP8_MAX
        scale[scale == 0] = 1.0
        q = (y / scale[:, None]).clamp(-_FP8_MAX, _FP8_MAX).to(torch.float8_e4m3fn)
        return [q.double(), scale, r]
    if op in ('conv', 'conv_train', 'conv_step'):
        K = case['K']
        step = op == 'conv_step'
        x = d['x'][:, None] if step else d['x']
        B, L, D = x.shape
        n = [L] * B if d.get('lengths') is None else d['lengths'].tolist()
        old = d['state'] if d['state'] is not None else x.new_zeros(B, K - 1, D)
        ys, lasts = [], []
        for b in range(B):   # one sequence at a time, a grouped convolution over what precedes and what is alive
            seq = torch.cat([old[b], x[b, :n[b]]]).t()
            lasts.append(seq[:, seq.shape[1] - (K - 1):].t())
            yb = F.silu(F.conv1d(seq[None], d['w'][:, None], d['b'], groups=D)[0].t()) if n[b] else x.new_zeros(0, D)
            ys.append(torch.cat([yb, x.new_zeros(L - n[b], D)]))
        y, last = torch.stack(ys), torch.stack(lasts)
        if step:
            return [y[:, 0], last]
        if not train:
            return [y, last] if case['carry'] else [y]
        if not case['carry']:
            return [y.detach(), *torch.autograd.grad(y, (d['x'], d['w'], d['b']), d['gy'])]
        gx, gw, gb, gs = torch.autograd.grad((y, last), (d['x'], d['w'], d['b'], d['state']), (d['gy'], d['gs']))
        return [y.detach(), gx, gw, gb, last.detach(), gs]
    step = op == 'scan_step'
    seq = (lambda t: t[:, None]) if step else (lambda t: t)
    u, raw, Bm, Cm = seq(d['u']), seq(d['dt']) + d['bias'], seq(d['Bm']), seq(d['Cm'])
    B, L, D = u.shape
    h = d['state'] if d['state'] is not None else u.new_zeros(B, D, case['N'])
    lengths = d.get('lengths')
    delta = F.softplus(raw, threshold=60.0)
    each = D // case['G']
    ys = []
    for dl, ut, bt, ct, t in zip(delta.unbind(1), u.unbind(1), Bm.unbind(1), Cm.unbind(1), range(L)):
        bt, ct = (m[:, :, None].expand(-1, -1, each, -1).reshape(B, D, -1) for m in (bt, ct))
        new = torch.exp(dl[..., None] * d['A']) * h + (dl * ut)[..., None] * bt
        yt = torch.einsum('bdn,bdn->bd', new, ct) + d['Dp'] * ut
        if lengths is not None:
            on = (lengths > t)[:, None]
            new, yt = torch.where(on[..., None], new, h), torch.where(on, yt, 0.0)
        h = new
        ys.append(yt)
    y = torch.stack(ys, 1)
    if case['gate']:
        y = y * F.silu(seq(d['z']))
    if step:
        return [y[:, 0], h]
    if not train:
        return [y, h] if case['carry'] else [y]
    leaves = [d[k] for k in ('u', 'dt', 'A', 'Bm', 'Cm', 'Dp', 'bias')] + ([d['z']] if case['gate'] else [])
    if not case['carry']:
        return [y.detach(), *torch.autograd.grad(y, leaves, d['gy'])]
    *grads, gs = torch.autograd.grad((y, h), leaves + [d['state']], (d['gy'], d['gs']))
    return [y.detach(), *grads, h.detach(), gs]
