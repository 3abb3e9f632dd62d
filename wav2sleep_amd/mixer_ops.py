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


_current_device = torch._C._cuda_getDevice if hasattr(torch._C, '_cuda_getDevice') else torch.cuda.current_device


class _On:
    """The tensors' device (an index) for the duration of a call; free where it is the current one already."""
    __slots__ = ('dev', 'ctx')

    def __init__(self, dev):
        self.dev, self.ctx = dev, None

    def __enter__(self):
        if _current_device() != self.dev:
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


def _match(ref, *wants) -> bool:
    """every (tensor or None, dtype, shape) is as wanted and on ref's device: the checks of a call in their quick form, without messages"""
    dev = ref.get_device()
    for t, dtype, shape in wants:
        if t is not None and (t.dtype is not dtype or t.shape != shape or t.get_device() != dev):
            return False
    return dev >= 0


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


def _opt_contig(*ts):
    return [t if t is None or t.is_contiguous() else t.contiguous() for t in ts]


# ------------------------------------------------------------------------------------------------------------------ short convolution
_ACT = {None: 0, 'linear': 0, 'silu': 1, 'swish': 1}


def _conv_args(x, weight, bias, act, state, lengths, y=None, state_out=None):
    ptr = lib.ptr
    B, L, D = x.shape
    sb, sl, _ = x.stride()
    return lib.ShortConvArgs(x.data_ptr(), ptr(state), weight.data_ptr(), ptr(bias), ptr(lengths), ptr(y), ptr(state_out), None, None, None, None, None, None, None,
                             sb, sl, 0, 0, B, L, D, weight.shape[1], lib.IO_DTYPES[x.dtype], act)


def _conv_forward(x, weight, bias, state, lengths, act, want_state):
    y = x.new_empty(x.shape)
    new = x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2])) if want_state else None
    lib.mixer_call('w2s_short_conv_fwd', _conv_args(x, weight, bias, act, state, lengths, y, new), x.get_device())
    return y, new


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, act, want_state):
        x = _cl(x)
        weight, bias, state = _opt_contig(weight, bias, state)
        with _On(x.get_device()):
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
        need = ctx.needs_input_grad
        dev = x.get_device()
        with _On(dev):
            gnew = None if gnew is None else gnew.contiguous()
            gx = x.new_empty(x.shape)
            gs = state.new_empty(state.shape) if need[3] else None
            if B == 0 or L == 0:   # no positions: nothing but the state's rows, which pass through
                if gs is not None:
                    gs.copy_(gnew) if gnew is not None else gs.zero_()
                return gx if need[0] else None, torch.zeros_like(weight) if need[1] else None, torch.zeros_like(bias) if need[2] else None, gs, None, None, None
            ptr = lib.ptr
            a = _conv_args(x, weight, bias, ctx.act, state, lengths)
            if gy is not None:
                gy = _cl(gy)
                a.gy = gy.data_ptr()
                a.sg_b, a.sg_l, _ = gy.stride()
            a.gstate, a.gx, a.gstate_in = ptr(gnew), gx.data_ptr(), ptr(gs)
            gw = gb = None
            if need[1] or need[2]:
                gw, gb = weight.new_empty(weight.shape), None if bias is None else bias.new_empty(bias.shape)
                part = weight.new_empty(lib.mixer_size('w2s_short_conv_part', a))
                a.gw, a.gbias, a.part = gw.data_ptr(), ptr(gb), part.data_ptr()
            lib.mixer_call('w2s_short_conv_bwd', a, dev)
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
    if not (isinstance(x, Tensor) and isinstance(weight, Tensor) and x.dim() == 3 and weight.dim() == 2 and 1 <= weight.shape[1] <= 8 and x.dtype in lib.IO_DTYPES
            and activation in _ACT and x.shape[2] >= 1
            and _match(x, (weight, _F32, (x.shape[2], weight.shape[1])), (bias, _F32, (x.shape[2],)),
                       (state, x.dtype, (x.shape[0], weight.shape[1] - 1, x.shape[2])), (lengths, torch.int32, (x.shape[0],)))):
        _io('x', x)
        if x.dim() != 3:
            raise ValueError(f'x: [B, L, D] expected, got {tuple(x.shape)}')
        _conv_check(x, weight, bias, activation)
        _like('state', state, x, (x.shape[0], weight.shape[1] - 1, x.shape[2]))
        _like('lengths', lengths, x, (x.shape[0],), torch.int32)
    if lengths is not None:
        lengths = lengths.contiguous()
    act = _ACT[activation]
    if _wants_grad(x, weight, bias, state):
        return _ShortConv.apply(x, weight, bias, state, lengths, act, bool(return_state))
    x = _cl(x)
    weight, bias, state = _opt_contig(weight, bias, state)
    with _On(x.get_device()):
        y, new = _conv_forward(x, weight, bias, state, lengths, act, return_state)
    return (y, new) if return_state else y


def short_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = 'silu',
                    state_out: Tensor | None = None) -> Tensor:
    """One position of `short_conv`: x [B, D], state [B, K-1, D] -> y [B, D].  The state moves on by one in place, or into state_out."""
    _no_grad_path('short_conv_step', x, state, weight, bias)
    if not (isinstance(x, Tensor) and isinstance(weight, Tensor) and isinstance(state, Tensor) and x.dim() == 2 and weight.dim() == 2 and 1 <= weight.shape[1] <= 8
            and x.dtype in lib.IO_DTYPES and activation in _ACT and x.shape[1] >= 1
            and _match(x, (weight, _F32, (x.shape[1], weight.shape[1])), (bias, _F32, (x.shape[1],)), (state, x.dtype, (x.shape[0], weight.shape[1] - 1, x.shape[1])))):
        _io('x', x)
        if x.dim() != 2:
            raise ValueError(f'x: [B, D] expected, got {tuple(x.shape)}')
        _conv_check(x, weight, bias, activation)
        if state is None:
            raise TypeError('state: a tensor is wanted')
        _like('state', state, x, (x.shape[0], weight.shape[1] - 1, x.shape[1]))
    out = _state_out(state, state_out)
    x = _cl(x)
    weight, bias = _opt_contig(weight, bias)
    y = x.new_empty(x.shape)
    dev = x.get_device()
    B, D = x.shape
    with _On(dev):
        lib.mixer_call('w2s_short_conv_step', lib.ShortConvArgs(x.data_ptr(), state.data_ptr(), weight.data_ptr(), lib.ptr(bias), None, y.data_ptr(), out.data_ptr(),
                                                                None, None, None, None, None, None, None, x.stride(0), 0, 0, 0, B, 1, D, weight.shape[1],
                                                                lib.IO_DTYPES[x.dtype], _ACT[activation]), dev)
    torch.autograd.graph.increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------------------------ selective scan
def _ssm_args(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, y=None, new=None, ckpt=None):
    ptr = lib.ptr
    nb, L, Dc = u.shape
    su, sd, sB, sC, sz = u.stride(), dt.stride(), B.stride(), C.stride(), (0, 0) if z is None else z.stride()
    return lib.SsmArgs(u.data_ptr(), dt.data_ptr(), ptr(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), ptr(D), ptr(dt_bias), ptr(state), ptr(lengths), ptr(y), ptr(new), ptr(ckpt),
                       None, None, None, None, None, None, None, None, None, None, None, None,
                       su[0], su[1], sd[0], sd[1], sz[0], sz[1], sB[0], sB[1], sB[2], sC[0], sC[1], sC[2], 0, 0,
                       nb, L, Dc, A.shape[1], B.shape[2], lib.IO_DTYPES[u.dtype], softplus, 0)


def _scan_forward(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, train):
    y = u.new_empty(u.shape)
    new = A.new_empty((u.shape[0], u.shape[2], A.shape[1])) if want_state else None
    a = _ssm_args(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, y, new)
    ckpt = None
    if train:
        ckpt = A.new_empty(lib.mixer_size('w2s_ssm_ckpt', a))
        a.ckpt = ckpt.data_ptr()
    n = lib.mixer_size('w2s_ssm_ws', a, 0)
    if n:
        ws = A.new_empty(n // 4)
        a.ws = ws.data_ptr()
    lib.mixer_call('w2s_ssm_scan_fwd', a, u.get_device())
    return y, new, ckpt


class _SsmScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state):
        u, dt, B, C, z = _cl(u), _cl(dt), _cl(B), _cl(C), _cl(z)
        A, D, dt_bias, state = _opt_contig(A, D, dt_bias, state)
        with _On(u.get_device()):
            y, new, ckpt = _scan_forward(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, True)
        ctx.save_for_backward(u, dt, A, B, C, D, z, dt_bias, state, lengths, ckpt)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return (y, new) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gnew=None):
        u, dt, A, B, C, D, z, dt_bias, state, lengths, ckpt = ctx.saved_tensors
        dev = u.get_device()
        with _On(dev):
            a = _ssm_args(u, dt, A, B, C, D, z, dt_bias, state, lengths, ctx.softplus, None, None, ckpt)
            if gnew is not None:
                gnew = gnew.contiguous()
                a.gh = gnew.data_ptr()
            if gy is not None:
                gy = _cl(gy)
                a.gy = gy.data_ptr()
                a.sg_b, a.sg_l, _ = gy.stride()
            new = lambda t: None if t is None else t.new_empty(t.shape)   # noqa: E731
            gu, gdt, gz, gB, gC, gA, gD, gbias, gs = out = [new(t) for t in (u, dt, z, B, C, A, D, dt_bias, state)]
            a.gu, a.gdt, a.gz, a.gB, a.gC, a.gA, a.gD, a.gbias, a.gh0 = [None if t is None else t.data_ptr() for t in out]
            ws = A.new_empty(max(1, lib.mixer_size('w2s_ssm_ws', a, 1) // 4))
            a.ws = ws.data_ptr()
            lib.mixer_call('w2s_ssm_scan_bwd', a, dev)
        return tuple([g if n else None for g, n in zip((gu, gdt, gA, gB, gC, gD, gz, gbias, gs), ctx.needs_input_grad)]) + (None, None, None)


def _ssm_check(u, dt, A, B, C, D, z, dt_bias, state, lengths, nrows):
    """-> B, C with their group dimension.  nrows: how many dimensions stand in front of the channels (2: sequences, 1: one position)"""
    if isinstance(u, Tensor) and isinstance(dt, Tensor) and isinstance(A, Tensor) and isinstance(B, Tensor) and isinstance(C, Tensor):
        if B.dim() == nrows + 1:
            B = B.unsqueeze(-2)
        if C.dim() == nrows + 1:
            C = C.unsqueeze(-2)
        shape, io = u.shape, u.dtype
        if u.dim() == nrows + 1 and A.dim() == 2 and B.dim() == nrows + 2 and io in lib.IO_DTYPES:
            rows, Dc, N, G = shape[:-1], shape[-1], A.shape[1], B.shape[-2]
            bc = (*rows, G, N)
            if 1 <= N <= 64 and Dc >= 1 and G >= 1 and Dc % G == 0 and _match(
                    u, (u, io, shape), (dt, io, shape), (z, io, shape), (A, _F32, (Dc, N)), (B, io, bc), (C, io, bc), (D, _F32, (Dc,)), (dt_bias, _F32, (Dc,)),
                    (state, _F32, (rows[0], Dc, N)), (lengths, torch.int32, rows[:1])):
                return B, C
    # something is wrong: say what
    _io('u', u)
    if u.dim() != nrows + 1:
        raise ValueError(f'u: {nrows + 1} dimensions expected, got {tuple(u.shape)}')
    rows, Dc = tuple(u.shape[:-1]), u.shape[-1]
    if dt is None or B is None or C is None or A is None:
        raise TypeError('dt, A, B and C: tensors are wanted')
    _like('dt', dt, u, u.shape)
    _like('z', z, u, u.shape)
    if not isinstance(A, Tensor) or A.dim() != 2 or A.shape[0] != Dc or not 1 <= A.shape[1] <= 64 or Dc < 1:
        raise ValueError(f'A: [{Dc}, N] with 1 <= N <= 64 expected, got {tuple(A.shape) if isinstance(A, Tensor) else A}')
    N = A.shape[1]
    _like('A', A, u, A.shape, _F32)
    _like('D', D, u, (Dc,), _F32)
    _like('dt_bias', dt_bias, u, (Dc,), _F32)
    G = B.shape[-2] if isinstance(B, Tensor) and B.dim() == nrows + 2 else 0
    if G < 1 or Dc % G:
        raise ValueError(f'B: {rows} + ([G,] {N}) with G a divisor of {Dc} expected, got {tuple(B.shape) if isinstance(B, Tensor) else B}')
    _like('B', B, u, rows + (G, N))
    _like('C', C, u, rows + (G, N))
    _like('state', state, u, (rows[0], Dc, N), _F32)
    _like('lengths', lengths, u, rows[:1], torch.int32)
    return B, C


def ssm_scan(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None, z: Tensor | None = None, dt_bias: Tensor | None = None,
             dt_softplus: bool = True, state: Tensor | None = None, lengths: Tensor | None = None, return_state: bool = False):
    """Selective state space scan.  With delta = softplus(dt + dt_bias) (dt_softplus=False: dt + dt_bias)

        h[b, t, d, n] = exp(delta A[d, n]) h[b, t-1, d, n] + delta u[b, t, d] B[b, t, g, n]
        y[b, t, d]    = (sum_n C[b, t, g, n] h[b, t, d, n] + D[d] u[b, t, d]) * silu(z[b, t, d])

    u, dt, z [B, L, D]; A [D, N], N <= 64 (negative for a stable scan); B, C [B, L, N] or [B, L, G, N]: channel d belongs to group d // (D / G);
    D, dt_bias [D].  state [B, D, N]: h in front of position 0 (None: zeros).  return_state: also h at the end, the `state` of a call that goes on."""
    B, C = _ssm_check(u, dt, A, B, C, D, z, dt_bias, state, lengths, 2)
    if lengths is not None:
        lengths = lengths.contiguous()
    if _wants_grad(u, dt, A, B, C, D, z, dt_bias, state):
        return _SsmScan.apply(u, dt, A, B, C, D, z, dt_bias, state, lengths, 1 if dt_softplus else 0, bool(return_state))
    A, D, dt_bias, state = _opt_contig(A, D, dt_bias, state)
    with _On(u.get_device()):
        y, new, _ = _scan_forward(_cl(u), _cl(dt), A, _cl(B), _cl(C), D, _cl(z), dt_bias, state, lengths, 1 if dt_softplus else 0, return_state, False)
    return (y, new) if return_state else y


def ssm_step(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None = None, z: Tensor | None = None,
             dt_bias: Tensor | None = None, dt_softplus: bool = True, state_out: Tensor | None = None) -> Tensor:
    """One position of `ssm_scan`: u, dt, z [B, D], B, C [B, N] or [B, G, N], state [B, D, N] fp32 -> y [B, D].  The state moves on in place, or
    into state_out."""
    _no_grad_path('ssm_step', u, dt, A, B, C, state, D, z, dt_bias)
    if state is None:
        raise TypeError('state: a tensor is wanted')
    B, C = _ssm_check(u, dt, A, B, C, D, z, dt_bias, state, None, 1)
    out = _state_out(state, state_out)
    u, dt, z, B, C = _cl(u), _cl(dt), _cl(z), _cl(B), _cl(C)
    A, D, dt_bias = _opt_contig(A, D, dt_bias)
    y = u.new_empty(u.shape)
    dev, ptr = u.get_device(), lib.ptr
    nb, Dc = u.shape
    sB, sC = B.stride(), C.stride()
    with _On(dev):
        lib.mixer_call('w2s_ssm_step', lib.SsmArgs(
            u.data_ptr(), dt.data_ptr(), ptr(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), ptr(D), ptr(dt_bias), state.data_ptr(), None, y.data_ptr(), out.data_ptr(), None,
            None, None, None, None, None, None, None, None, None, None, None, None,
            u.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0), 0, sB[0], 0, sB[1], sC[0], 0, sC[1], 0, 0,
            nb, 1, Dc, A.shape[1], B.shape[1], lib.IO_DTYPES[u.dtype], 1 if dt_softplus else 0, 0), dev)
    torch.autograd.graph.increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------------------------ norm with the residual's addition
def _rows(t, C):
    """t as [rows, C] with contiguous rows (a view where its strides allow one)"""
    return None if t is None else _cl(t).reshape(-1, C)


def _norm_forward(x, weight, residual, eps, fp8, want_rstd):
    shape, C = x.shape, x.shape[-1]
    x2, r2 = _rows(x, C), _rows(residual, C)
    rows, code = x2.shape[0], lib.IO_DTYPES[x.dtype]
    y = x.new_empty(shape, dtype=torch.float8_e4m3fn) if fp8 else x.new_empty(shape)
    r = None if residual is None else residual.new_empty(shape)
    scale = weight.new_empty(shape[:-1]) if fp8 else None
    rstd = weight.new_empty(rows) if want_rstd else None
    ptr = lib.ptr
    a = lib.AddNormArgs(x2.data_ptr(), ptr(r2), weight.data_ptr(), y.data_ptr(), ptr(r), ptr(scale), ptr(rstd), None, None, None, None, None, None,
                        rows, x2.stride(0), 0 if r2 is None else r2.stride(0), 0, 0, C, code, code if residual is None else lib.IO_DTYPES[residual.dtype], int(fp8), eps, 0)
    lib.mixer_call('w2s_add_norm_fwd', a, x.get_device())
    return y, r, scale, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        weight, = _opt_contig(weight)
        with _On(x.get_device()):
            y, r, _, rstd = _norm_forward(x, weight, residual, eps, False, True)
        # the backward needs the sum as it was normalised: r where that is exact (fp32), else the two addends again
        if r is not None and r.dtype == _F32:
            ctx.save_for_backward(None, r, weight, rstd)
        else:
            ctx.save_for_backward(x, residual, weight, rstd)
        ctx.x_dtype, ctx.eps = x.dtype, eps
        ctx.set_materialize_grads(False)
        return (y, r) if r is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gr=None):
        x, res, weight, rstd = ctx.saved_tensors
        first = res if x is None else x
        shape, C, dev = first.shape, first.shape[-1], first.get_device()
        need, xt = ctx.needs_input_grad, ctx.x_dtype
        rtype = res.dtype if res is not None else xt
        with _On(dev):
            ptr = lib.ptr
            x2, r2, gy2, gr2 = _rows(x, C), _rows(res, C), _rows(gy, C), _rows(gr, C)
            gx = first.new_empty(shape, dtype=xt) if need[0] or (need[2] and rtype is xt) else None
            gres = first.new_empty(shape, dtype=rtype) if need[2] and rtype is not xt else None
            ld = lambda t: 0 if t is None else t.stride(0)   # noqa: E731
            a = lib.AddNormArgs(ptr(x2), ptr(r2), weight.data_ptr(), None, None, None, rstd.data_ptr(), ptr(gy2), ptr(gr2), ptr(gx), ptr(gres), None, None,
                                rstd.shape[0], ld(x2), ld(r2), ld(gy2), ld(gr2), C, lib.IO_DTYPES[xt], lib.IO_DTYPES[rtype], 0, ctx.eps, 0)
            gw = None
            if need[1]:
                gw = weight.new_empty(weight.shape)
                part = weight.new_empty(lib.mixer_size('w2s_add_norm_part', a))
                a.gw, a.part = gw.data_ptr(), part.data_ptr()
            lib.mixer_call('w2s_add_norm_bwd', a, dev)
        both = gx if gres is None else gres   # of one type, both addends have the same gradient
        return gx if need[0] else None, gw, both if need[2] else None, None


def _norm_check(x, weight, residual, eps):
    if (isinstance(x, Tensor) and isinstance(weight, Tensor) and x.dtype in lib.IO_DTYPES and x.dim() >= 1 and x.shape[-1] >= 1 and eps >= 0.0
            and (residual is None or isinstance(residual, Tensor) and residual.dtype in (x.dtype, _F32))
            and _match(x, (weight, _F32, x.shape[-1:]), (residual, None if residual is None else residual.dtype, x.shape))):
        return
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
    weight, = _opt_contig(weight)
    with _On(x.get_device()):
        y, r, _, _ = _norm_forward(x, weight, residual, float(eps), False, False)
    return y, (x if r is None else r)


def add_rms_norm_8bit(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-5):
    """`add_rms_norm` with y in 8 bits: returns (q, scale, r), q float8_e4m3fn of x's shape, scale fp32 [...] with y ~ q * scale[..., None] -- the row-wise
    scaled operand of an 8-bit matrix product.  scale = max|y| / 448 over the row (1 for a row of zeros; NaN where the row holds one).  No backward."""
    _norm_check(x, weight, residual, eps)
    _no_grad_path('add_rms_norm_8bit', x, weight, residual)
    weight, = _opt_contig(weight)
    with _On(x.get_device()):
        q, r, scale, _ = _norm_forward(x, weight, residual, float(eps), True, False)
    return q, scale, (x if r is None else r)
