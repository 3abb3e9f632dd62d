"""Operators of a causal state space sequence mixer, as functions on device tensors (kernels: csrc/short_conv.hip, ssm_scan.hip, add_norm.hip).

    y          = short_conv(x, weight, bias)             depthwise causal convolution of up to 8 taps (+ SiLU)
    y          = ssm_scan(u, dt, A, B, C, D, z, dt_bias) selective state space scan (+ gate)
    y, r       = add_rms_norm(x, weight, residual)       r = x + residual, y = RMS norm of r
    q, s, r    = add_rms_norm_8bit(x, weight, residual)  the same with y in 8 bits (e4m3) and a scale per row
    y          = short_conv_step(...) / ssm_step(...)    one position of a stream: the state goes in and comes out

They are what `SequenceSSM` runs on; the reference mixes epochs with dilated convolutions only (models/wav2sleep.py:349-390).  The first three are
differentiable (first order) in every floating argument.  Activations are fp32, bf16 or fp16, all of one type in a call, channels last, with any
strides in front of a contiguous channel dimension (a tensor with another channel stride is copied first); results are contiguous.  Parameters and the
scan's states are fp32.  Arithmetic is fp32; a 16-bit result is rounded once.  Everything runs on the current stream of the tensors' device,
allocates from torch's allocator, never synchronises, and records into a hipGraph.  CPU tensors raise (lib.W2SError): there is no CPU path.

lengths (int32 [B], on the device): sequence b ends in front of position lengths[b], clamped to [0, L].  Inputs at and behind the end are not read,
results and gradients there are 0, and a returned state is the one at the end (the initial state for a length of 0).
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import lib

_F32 = torch.float32


class _On:
    """The tensors' device for the duration of a call; free where it is the current one already."""
    __slots__ = ('dev', 'ctx')

    def __init__(self, dev):
        self.dev, self.ctx = dev, None

    def __enter__(self):
        if torch.cuda.current_device() != self.dev.index:
            self.ctx = torch.cuda.device(self.dev)
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)


def _cl(t):
    """t with a contiguous last dimension"""
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _io(name, t):
    if not isinstance(t, Tensor):
        raise TypeError(f'{name}: a tensor is wanted, got {type(t).__name__}')
    if not t.is_cuda:
        raise lib.W2SError(f'{name}: wav2sleep_amd kernels need device tensors (no CPU path)')
    if t.dtype not in lib.IO_DTYPES:
        raise ValueError(f'{name}: float32, bfloat16 or float16 expected, got {t.dtype}')


def _like(name, t, ref, shape, dtype=None):
    """optional tensor `t` has this shape, ref's device and the type `dtype` (ref's when None)"""
    if t is None:
        return
    if not isinstance(t, Tensor):
        raise TypeError(f'{name}: a tensor is wanted, got {type(t).__name__}')
    if t.device != ref.device:
        raise lib.W2SError(f'{name}: on {t.device}, the other tensors are on {ref.device}')
    want = ref.dtype if dtype is None else dtype
    if t.dtype != want:
        raise ValueError(f'{name}: {want} expected, got {t.dtype}')
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name}: shape {tuple(shape)} expected, got {tuple(t.shape)}')


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _no_grad_path(what, *ts):
    if _wants_grad(*ts):
        raise lib.W2SError(f'{what} has no backward: call it under torch.no_grad() or detach its arguments')


def _state_out(state, state_out):
    """where a step leaves its state: `state` itself unless another tensor is given"""
    if state_out is None:
        state_out = state
    else:
        _like('state_out', state_out, state, state.shape)
        a, b, n = state.data_ptr(), state_out.data_ptr(), state.numel() * state.element_size()
        if a != b and a < b + n and b < a + n:
            raise ValueError('state_out overlaps state without being the same tensor')
    if not state_out.is_contiguous() or not state.is_contiguous():
        raise ValueError('state / state_out of a step must be contiguous')
    if state_out.requires_grad:
        raise lib.W2SError('state_out requires a gradient: a step overwrites it')
    return state_out


# ------------------------------------------------------------------------------------------------------------------ short convolution
_ACT = {None: 0, 'linear': 0, 'silu': 1, 'swish': 1}


def _conv_args(x, weight, bias, act, state, lengths):
    a = lib.ShortConvArgs()
    ptr = lib.ptr
    a.x, a.state, a.w, a.bias, a.lengths = ptr(x), ptr(state), ptr(weight), ptr(bias), ptr(lengths)
    a.B, a.L, a.D = x.shape
    a.K, a.dtype, a.act = weight.shape[1], lib.IO_DTYPES[x.dtype], act
    a.sx_b, a.sx_l = x.stride(0), x.stride(1)
    return a


def _conv_forward(x, weight, bias, state, lengths, act, want_state):
    a = _conv_args(x, weight, bias, act, state, lengths)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    new = torch.empty(x.shape[0], a.K - 1, x.shape[2], device=x.device, dtype=x.dtype) if want_state else None
    a.y, a.state_out = lib.ptr(y), lib.ptr(new)
    lib.mixer_call('w2s_short_conv_fwd', a)
    return y, new


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, act, want_state):
        x, weight, bias, state = _cl(x), weight.contiguous(), None if bias is None else bias.contiguous(), None if state is None else state.contiguous()
        with _On(x.device):
            y, new = _conv_forward(x, weight, bias, state, lengths, act, want_state)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return (y, new) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gnew=None):
        x, weight, bias, state, lengths = ctx.saved_tensors
        B, L, D = x.shape
        K = weight.shape[1]
        need = ctx.needs_input_grad
        with _On(x.device):
            gy, gnew = _cl(gy), None if gnew is None else gnew.contiguous()
            gx = torch.empty(B, L, D, device=x.device, dtype=x.dtype)
            gs = torch.empty_like(state) if state is not None and need[3] else None
            if B == 0 or L == 0:   # no positions: nothing but the state's rows, which pass through
                gw, gb = torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias)
                if gs is not None:
                    gs.copy_(gnew) if gnew is not None else gs.zero_()
                return gx if need[0] else None, gw, gb, gs, None, None, None
            a = _conv_args(x, weight, bias, ctx.act, state, lengths)
            a.gy, a.gstate, a.gx, a.gstate_in = lib.ptr(gy), lib.ptr(gnew), lib.ptr(gx), lib.ptr(gs)
            if gy is not None:
                a.sg_b, a.sg_l = gy.stride(0), gy.stride(1)
            gw = gb = part = None
            if need[1] or need[2]:
                gw = torch.empty_like(weight)
                gb = torch.empty_like(bias) if bias is not None else None
                part = torch.empty(lib.mixer_size('w2s_short_conv_part', a), device=x.device, dtype=_F32)
                a.gw, a.gbias, a.part = lib.ptr(gw), lib.ptr(gb), lib.ptr(part)
            lib.mixer_call('w2s_short_conv_bwd', a)
        return gx if need[0] else None, gw if need[1] else None, gb if need[2] else None, gs, None, None, None


def _conv_check(x, weight, bias, activation):
    _io('x', x)
    if activation not in _ACT:
        raise ValueError(f'{activation=} is unsupported (one of {list(_ACT)})')
    D = x.shape[-1]
    if not isinstance(weight, Tensor) or weight.dim() != 2 or weight.shape[0] != D or not 1 <= weight.shape[1] <= 8:
        raise ValueError(f'weight: [{D}, K] with 1 <= K <= 8 expected, got {tuple(weight.shape) if isinstance(weight, Tensor) else weight}')
    if D < 1:
        raise ValueError('x has no channels')
    _like('weight', weight, x, weight.shape, _F32)
    _like('bias', bias, x, (D,), _F32)


def short_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = 'silu', state: Tensor | None = None,
               lengths: Tensor | None = None, return_state: bool = False):
    """Depthwise causal convolution: y[b, t, d] = act(bias[d] + sum_k weight[d, k] x[b, t - (K-1) + k, d]).

    x [B, L, D]; weight [D, K], K <= 8; activation 'silu' or None.  state [B, K-1, D] (x's type): the inputs in front of position 0, oldest first
    (None: zeros).  return_state: also the last K-1 inputs, the `state` of a call that goes on (from `state` itself where a sequence is shorter)."""
    _io('x', x)
    if x.dim() != 3:
        raise ValueError(f'x: [B, L, D] expected, got {tuple(x.shape)}')
    _conv_check(x, weight, bias, activation)
    B, _, D = x.shape
    _like('state', state, x, (B, weight.shape[1] - 1, D))
    _like('lengths', lengths, x, (B,), torch.int32)
    if lengths is not None:
        lengths = lengths.contiguous()
    act = _ACT[activation]
    if _wants_grad(x, weight, bias, state):
        return _ShortConv.apply(x, weight, bias, state, lengths, act, bool(return_state))
    with _On(x.device):
        y, new = _conv_forward(_cl(x), weight.contiguous(), None if bias is None else bias.contiguous(), None if state is None else state.contiguous(), lengths,
                               act, return_state)
    return (y, new) if return_state else y


def short_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = 'silu',
                    state_out: Tensor | None = None) -> Tensor:
    """One position of `short_conv`: x [B, D], state [B, K-1, D] -> y [B, D].  The state moves on by one in place, or into state_out."""
    _no_grad_path('short_conv_step', x, state, weight, bias)
    _io('x', x)
    if x.dim() != 2:
        raise ValueError(f'x: [B, D] expected, got {tuple(x.shape)}')
    _conv_check(x, weight, bias, activation)
    _like('state', state, x, (x.shape[0], weight.shape[1] - 1, x.shape[1]))
    out = _state_out(state, state_out)
    with _On(x.device):
        x = _cl(x)
        weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        a = lib.ShortConvArgs()
        ptr = lib.ptr
        a.x, a.state, a.w, a.bias, a.y, a.state_out = ptr(x), ptr(state), ptr(weight), ptr(bias), ptr(y), ptr(out)
        a.B, a.L, a.D, a.K, a.dtype, a.act, a.sx_b = x.shape[0], 1, x.shape[1], weight.shape[1], lib.IO_DTYPES[x.dtype], _ACT[activation], x.stride(0)
        lib.mixer_call('w2s_short_conv_step', a)
    torch.autograd.graph.increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------------------------ selective scan
def _ssm_args(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus):
    a = lib.SsmArgs()
    ptr = lib.ptr
    a.u, a.dt, a.z, a.Bm, a.Cm = ptr(u), ptr(dt), ptr(z), ptr(B), ptr(C)
    a.A, a.Dp, a.dt_bias, a.h0, a.lengths = ptr(A), ptr(D), ptr(dt_bias), ptr(state), ptr(lengths)
    a.B, a.L, a.D = u.shape
    a.N, a.G, a.dtype, a.softplus = A.shape[1], B.shape[2], lib.IO_DTYPES[u.dtype], int(softplus)
    a.su_b, a.su_l, _ = u.stride()
    a.sdt_b, a.sdt_l, _ = dt.stride()
    if z is not None:
        a.sz_b, a.sz_l, _ = z.stride()
    a.sB_b, a.sB_l, a.sB_g, _ = B.stride()
    a.sC_b, a.sC_l, a.sC_g, _ = C.stride()
    return a


def _scan_forward(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, train):
    a = _ssm_args(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus)
    y = torch.empty(u.shape, device=u.device, dtype=u.dtype)
    new = torch.empty(u.shape[0], u.shape[2], a.N, device=u.device, dtype=_F32) if want_state else None
    ckpt = None
    if train:
        ckpt = torch.empty(lib.mixer_size('w2s_ssm_ckpt', a), device=u.device, dtype=_F32)
        a.ckpt = lib.ptr(ckpt)
    n = lib.mixer_size('w2s_ssm_ws', a, 0)
    ws = torch.empty(n, device=u.device, dtype=torch.uint8) if n else None
    a.y, a.h_out, a.ws = lib.ptr(y), lib.ptr(new), lib.ptr(ws)
    lib.mixer_call('w2s_ssm_scan_fwd', a)
    return y, new, ckpt


def _opt_contig(*ts):
    return tuple(None if t is None else t.contiguous() for t in ts)


class _SsmScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state):
        u, dt, B, C, z = _cl(u), _cl(dt), _cl(B), _cl(C), _cl(z)
        A, D, dt_bias, state = _opt_contig(A, D, dt_bias, state)
        with _On(u.device):
            y, new, ckpt = _scan_forward(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, True)
        ctx.save_for_backward(u, dt, A, B, C, D, z, dt_bias, state, lengths, ckpt)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return (y, new) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gnew=None):
        u, dt, A, B, C, D, z, dt_bias, state, lengths, ckpt = ctx.saved_tensors
        dev, io = u.device, u.dtype
        with _On(dev):
            gy, gnew = _cl(gy), None if gnew is None else gnew.contiguous()
            a = _ssm_args(u, dt, A, B, C, D, z, dt_bias, state, lengths, ctx.softplus)
            new = lambda t, dtype=io: None if t is None else torch.empty(t.shape, device=dev, dtype=dtype)   # noqa: E731
            gu, gdt, gz, gB, gC = new(u), new(dt), new(z), new(B), new(C)
            gA, gD, gbias, gs = new(A, _F32), new(D, _F32), new(dt_bias, _F32), new(state, _F32)
            ptr = lib.ptr
            a.gy, a.gh, a.ckpt = ptr(gy), ptr(gnew), ptr(ckpt)
            if gy is not None:
                a.sg_b, a.sg_l, _ = gy.stride()
            a.gu, a.gdt, a.gz, a.gB, a.gC, a.gA, a.gD, a.gbias, a.gh0 = (ptr(t) for t in (gu, gdt, gz, gB, gC, gA, gD, gbias, gs))
            ws = torch.empty(max(1, lib.mixer_size('w2s_ssm_ws', a, 1)), device=dev, dtype=torch.uint8)
            a.ws = ptr(ws)
            lib.mixer_call('w2s_ssm_scan_bwd', a)
        out = [gu, gdt, gA, gB, gC, gD, gz, gbias, gs]
        return tuple(g if n else None for g, n in zip(out, ctx.needs_input_grad)) + (None, None, None)


def _ssm_check(u, dt, A, B, C, D, z, dt_bias, rows):
    _io('u', u)
    if u.dim() != len(rows) + 1:
        raise ValueError(f'u: {len(rows) + 1} dimensions expected, got {tuple(u.shape)}')
    rows, Dc = tuple(u.shape[:-1]), u.shape[-1]
    _like('dt', dt, u, u.shape)
    _like('z', z, u, u.shape)
    if not isinstance(A, Tensor) or A.dim() != 2 or A.shape[0] != Dc or not 1 <= A.shape[1] <= 64 or Dc < 1:
        raise ValueError(f'A: [{Dc}, N] with 1 <= N <= 64 expected, got {tuple(A.shape) if isinstance(A, Tensor) else A}')
    N = A.shape[1]
    _like('A', A, u, A.shape, _F32)
    _like('D', D, u, (Dc,), _F32)
    _like('dt_bias', dt_bias, u, (Dc,), _F32)
    if not isinstance(B, Tensor) or not isinstance(C, Tensor):
        raise TypeError('B and C: tensors are wanted')
    if B.dim() == len(rows) + 1:
        B = B.unsqueeze(-2)
    if C.dim() == len(rows) + 1:
        C = C.unsqueeze(-2)
    G = B.shape[-2] if B.dim() == len(rows) + 2 else 0
    if G < 1 or Dc % G:
        raise ValueError(f'B: {rows} + ([G,] {N}) with G a divisor of {Dc} expected, got {tuple(B.shape)}')
    _like('B', B, u, rows + (G, N))
    _like('C', C, u, rows + (G, N))
    if dt is None:
        raise TypeError('dt: a tensor is wanted')
    return B, C


def ssm_scan(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None, z: Tensor | None = None, dt_bias: Tensor | None = None,
             dt_softplus: bool = True, state: Tensor | None = None, lengths: Tensor | None = None, return_state: bool = False):
    """Selective state space scan.  With delta = softplus(dt + dt_bias) (dt_softplus=False: dt + dt_bias)

        h[b, t, d, n] = exp(delta A[d, n]) h[b, t-1, d, n] + delta u[b, t, d] B[b, t, g, n]
        y[b, t, d]    = (sum_n C[b, t, g, n] h[b, t, d, n] + D[d] u[b, t, d]) * silu(z[b, t, d])

    u, dt, z [B, L, D]; A [D, N], N <= 64 (negative for a stable scan); B, C [B, L, N] or [B, L, G, N]: channel d belongs to group d // (D / G);
    D, dt_bias [D].  state [B, D, N]: h in front of position 0 (None: zeros).  return_state: also h at the end, the `state` of a call that goes on."""
    B, C = _ssm_check(u, dt, A, B, C, D, z, dt_bias, (0, 0))
    nb, _, Dc = u.shape
    _like('state', state, u, (nb, Dc, A.shape[1]), _F32)
    _like('lengths', lengths, u, (nb,), torch.int32)
    if lengths is not None:
        lengths = lengths.contiguous()
    if _wants_grad(u, dt, A, B, C, D, z, dt_bias, state):
        return _SsmScan.apply(u, dt, A, B, C, D, z, dt_bias, state, lengths, bool(dt_softplus), bool(return_state))
    A, D, dt_bias, state = _opt_contig(A, D, dt_bias, state)
    with _On(u.device):
        y, new, _ = _scan_forward(_cl(u), _cl(dt), A, _cl(B), _cl(C), D, _cl(z), dt_bias, state, lengths, dt_softplus, return_state, False)
    return (y, new) if return_state else y


def ssm_step(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None = None, z: Tensor | None = None,
             dt_bias: Tensor | None = None, dt_softplus: bool = True, state_out: Tensor | None = None) -> Tensor:
    """One position of `ssm_scan`: u, dt, z [B, D], B, C [B, N] or [B, G, N], state [B, D, N] fp32 -> y [B, D].  The state moves on in place, or
    into state_out."""
    _no_grad_path('ssm_step', u, dt, A, B, C, state, D, z, dt_bias)
    B, C = _ssm_check(u, dt, A, B, C, D, z, dt_bias, (0,))
    _like('state', state, u, (u.shape[0], u.shape[1], A.shape[1]), _F32)
    if state is None:
        raise TypeError('state: a tensor is wanted')
    out = _state_out(state, state_out)
    with _On(u.device):
        u, dt, z, B, C = _cl(u), _cl(dt), _cl(z), _cl(B), _cl(C)
        A, D, dt_bias = _opt_contig(A, D, dt_bias)
        y = torch.empty(u.shape, device=u.device, dtype=u.dtype)
        a = lib.SsmArgs()
        ptr = lib.ptr
        a.u, a.dt, a.z, a.Bm, a.Cm, a.A, a.Dp, a.dt_bias, a.h0, a.y, a.h_out = (ptr(t) for t in (u, dt, z, B, C, A, D, dt_bias, state, y, out))
        a.B, a.L, a.D, a.N, a.G, a.dtype, a.softplus = u.shape[0], 1, u.shape[1], A.shape[1], B.shape[1], lib.IO_DTYPES[u.dtype], int(bool(dt_softplus))
        a.su_b, a.sdt_b = u.stride(0), dt.stride(0)
        if z is not None:
            a.sz_b = z.stride(0)
        a.sB_b, a.sB_g, _ = B.stride()
        a.sC_b, a.sC_g, _ = C.stride()
        lib.mixer_call('w2s_ssm_step', a)
    torch.autograd.graph.increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------------------------ norm with the residual's addition
def _rows(t, C):
    """t as [rows, C] with contiguous rows (a view where its strides allow one)"""
    return None if t is None else _cl(t).reshape(-1, C)


def _norm_forward(x, weight, residual, eps, fp8, want_rstd):
    C = x.shape[-1]
    x2, r2 = _rows(x, C), _rows(residual, C)
    a = lib.AddNormArgs()
    ptr = lib.ptr
    dev = x.device
    a.rows, a.C, a.dtype, a.eps, a.fp8 = x2.shape[0], C, lib.IO_DTYPES[x.dtype], eps, int(fp8)
    a.ldx, a.rdtype = x2.stride(0), a.dtype
    y = torch.empty(x.shape, device=dev, dtype=torch.float8_e4m3fn if fp8 else x.dtype)
    r = scale = rstd = None
    if residual is not None:
        r = torch.empty(x.shape, device=dev, dtype=residual.dtype)
        a.res, a.r, a.ldres, a.rdtype = ptr(r2), ptr(r), r2.stride(0), lib.IO_DTYPES[residual.dtype]
    if fp8:
        scale = torch.empty(x.shape[:-1], device=dev, dtype=_F32)
    if want_rstd:
        rstd = torch.empty(x2.shape[0], device=dev, dtype=_F32)
    a.x, a.w, a.y, a.scale, a.rstd = ptr(x2), ptr(weight), ptr(y), ptr(scale), ptr(rstd)
    lib.mixer_call('w2s_add_norm_fwd', a)
    return y, r, scale, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        weight = weight.contiguous()
        with _On(x.device):
            y, r, _, rstd = _norm_forward(x, weight, residual, eps, False, True)
        # the backward needs the sum as it was normalised: r where that is exact (fp32), else the two addends again
        if r is not None and r.dtype == _F32:
            ctx.save_for_backward(None, r, weight, rstd)
        else:
            ctx.save_for_backward(x, residual, weight, rstd)
        ctx.x_dtype, ctx.eps, ctx.joined = x.dtype, eps, residual is not None
        ctx.set_materialize_grads(False)
        return (y, r) if r is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gr=None):
        x, res, weight, rstd = ctx.saved_tensors
        first = res if x is None else x
        shape, C, dev = first.shape, first.shape[-1], first.device
        need = ctx.needs_input_grad
        rtype = res.dtype if res is not None else ctx.x_dtype
        with _On(dev):
            ptr = lib.ptr
            a = lib.AddNormArgs()
            a.C, a.dtype, a.rdtype, a.eps = C, lib.IO_DTYPES[ctx.x_dtype], lib.IO_DTYPES[rtype], ctx.eps
            keep = [_rows(t, C) for t in (x, res, gy, gr)]
            a.rows = rstd.shape[0]
            for (p, ld), t in zip((('x', 'ldx'), ('res', 'ldres'), ('gy', 'ldgy'), ('gr', 'ldgr')), keep):
                if t is not None:
                    setattr(a, p, ptr(t))
                    setattr(a, ld, t.stride(0))
            gx = torch.empty(shape, device=dev, dtype=ctx.x_dtype) if need[0] or (need[2] and rtype == ctx.x_dtype) else None
            gres = torch.empty(shape, device=dev, dtype=rtype) if need[2] and rtype != ctx.x_dtype else None
            a.w, a.rstd, a.gx, a.gres = ptr(weight), ptr(rstd), ptr(gx), ptr(gres)
            gw = None
            if need[1]:
                gw = torch.empty_like(weight)
                part = torch.empty(lib.mixer_size('w2s_add_norm_part', a), device=dev, dtype=_F32)
                a.gw, a.part = ptr(gw), ptr(part)
            lib.mixer_call('w2s_add_norm_bwd', a)
        both = gx if gres is None else gres   # of one type, both addends have the same gradient
        return gx if need[0] else None, gw, both if need[2] else None, None


def _norm_check(x, weight, residual, eps):
    _io('x', x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'x: [..., C] expected, got {tuple(x.shape)}')
    _like('weight', weight, x, (x.shape[-1],), _F32)
    if weight is None:
        raise TypeError('weight: a tensor is wanted')
    if residual is not None:
        _like('residual', residual, x, x.shape, _F32 if isinstance(residual, Tensor) and residual.dtype == _F32 else x.dtype)
    if not eps >= 0.0:
        raise ValueError(f'{eps=}: not negative')


def add_rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-5):
    """r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight over the last dimension; returns (y, r).  residual: x's type or fp32 (a residual stream
    in 32 bits), which is r's type; y has x's.  The sum is fp32 and y comes from it before r is rounded.  residual=None: r is x itself."""
    _norm_check(x, weight, residual, eps)
    if _wants_grad(x, weight, residual):
        out = _AddRmsNorm.apply(x, weight, residual, float(eps))
        return out if residual is not None else (out, x)
    with _On(x.device):
        y, r, _, _ = _norm_forward(x, weight.contiguous(), residual, float(eps), False, False)
    return y, (x if r is None else r)


def add_rms_norm_8bit(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-5):
    """`add_rms_norm` with y in 8 bits: returns (q, scale, r), q float8_e4m3fn of x's shape, scale fp32 [...] with y ~ q * scale[..., None] -- the row-wise
    scaled operand of an 8-bit matrix product.  scale = max|y| / 448 over the row (1 for a row of zeros; NaN where the row holds one).  No backward."""
    _norm_check(x, weight, residual, eps)
    _no_grad_path('add_rms_norm_8bit', x, weight, residual)
    with _On(x.device):
        q, r, scale, _ = _norm_forward(x, weight.contiguous(), residual, float(eps), True, False)
    return q, scale, (x if r is None else r)
