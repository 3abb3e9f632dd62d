"""Operators of a causal state space sequence mixer, as functions on device tensors (kernels: csrc/short_conv.hip, ssm_scan.hip, add_norm.hip).

    y          = short_conv(x, weight, bias)             depthwise causal convolution of up to 8 taps (+ SiLU)
    y          = ssm_scan(u, dt, A, B, C, D, z, dt_bias) selective state space scan (+ gate)
    y, r       = add_rms_norm(x, weight, residual)       r = x + residual, y = RMS norm of r
    q, s, r    = add_rms_norm_8bit(x, weight, residual)  the same with y in 8 bits (e4m3) and a scale per row
    y          = short_conv_step(...) / ssm_step(...)    one position of a stream: the state goes in and comes out

They are what `SequenceSSM` runs on; the reference mixes epochs with dilated convolutions only (models/wav2sleep.py:349-390).  The first three are
differentiable in every floating argument: in reverse mode, first order (a second one raises), and not in forward mode (an argument or an arriving gradient
with a tangent raises, in all six).  Activations are fp32, bf16 or fp16, all of one type in a call, channels last, with any strides in front of a contiguous
channel dimension (a tensor with another channel stride is copied first; the scan's positions lie less than 2^22 elements apart); results are contiguous.
Sizes go up to 2^30 and a launch has fewer than 2^32 threads; a call beyond that raises.  Parameters and the scan's states are fp32.  Arithmetic is fp32; a
16-bit result is rounded once.  Everything runs on the current stream of the tensors' device, allocates from torch's allocator, never synchronises, and
records into a hipGraph.  CPU tensors raise (lib.W2SError): there is no CPU path.

lengths (int32 [B], on the device): sequence b ends in front of position lengths[b], clamped to [0, L].  What the inputs hold at and behind the end, NaN
too, has no part in anything (the memory has to be there: a tile's loads run on to L); results and gradients there are 0, and a returned state is the one at
the end (the initial state for a length of 0).

A scan's backward takes scratch memory of 8 n bytes a position and block of 16 channels of a group, n being N rounded up to 8, 16, 32 or 64 (n / 2 bytes a
position and channel where groups fill their blocks; 8 n for groups of a single channel), and its forward keeps n floats a channel every 32 or 64 positions.
A backward that a hipGraph captures wants leaves that no living eager graph of the default stream holds (detached ones will do), and raises otherwise.
jit.trace, make_fx and export raise; torch.compile calls the operators between its graphs.  No other argument of a step may overlap its `state_out`.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import lib

_F32 = torch.float32
_ext = None


def _ops():
    """csrc/torch_ops.cpp: checks, allocation, launch and autograd node of a call, without the interpreter; None from it means a wrong argument"""
    global _ext
    if _ext is None:
        _ext = lib.load_torch_ops()
    return _ext


# ------------------------------------------------------------------------------------------------------------------ what is wrong with a refused call
def _sizes(name, t):
    if any(n > 1 << 30 for n in t.shape):
        raise ValueError(f'{name}: sizes up to 2^30 expected, got {tuple(t.shape)}')


def no_trace(what):
    if _ops().traced():
        raise lib.W2SError(f'{what}: no tracing here, a trace would hold results without their values')


def _io(name, t):
    if not isinstance(t, Tensor):
        raise TypeError(f'{name}: a tensor is wanted, got {type(t).__name__}')
    if not t.is_cuda:
        raise lib.W2SError(f'{name}: wav2sleep_amd kernels need device tensors (no CPU path)')
    no_trace(name)   # (in front of the checks of shapes, which a trace would record)
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


def _no_grad_path(what, *ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise lib.W2SError(f'{what} has no backward: call it under torch.no_grad() or detach its arguments')


def _state_check(state, state_out):
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


def no_forward_mode(what, *ts):
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise lib.W2SError(f'{what} has no forward-mode derivative: an argument carries a tangent')


def _refused(what, *ts):
    no_forward_mode(what, *ts)
    raise lib.W2SError(f'{what}: arguments refused (dense tensors are wanted)')


def _conv_check(x, weight, bias, activation):
    _io('x', x)
    _sizes('x', x)
    if activation not in _ACT:
        raise ValueError(f'{activation=} is unsupported (one of {list(_ACT)})')
    D = x.shape[-1]
    if not isinstance(weight, Tensor) or weight.dim() != 2 or weight.shape[0] != D or not 1 <= weight.shape[1] <= 8:
        raise ValueError(f'weight: [{D}, K] with 1 <= K <= 8 expected, got {tuple(weight.shape) if isinstance(weight, Tensor) else weight}')
    if D < 1:
        raise ValueError('x has no channels')
    _like('weight', weight, x, weight.shape, _F32)
    _like('bias', bias, x, (D,), _F32)


def _ssm_check(u, dt, A, B, C, D, z, dt_bias, state, lengths, nrows):
    """nrows: how many dimensions stand in front of the channels (2: sequences, 1: one position)"""
    _io('u', u)
    if u.dim() != nrows + 1:
        raise ValueError(f'u: {nrows + 1} dimensions expected, got {tuple(u.shape)}')
    _sizes('u', u)
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
    B, C = (t.unsqueeze(-2) if isinstance(t, Tensor) and t.dim() == nrows + 1 else t for t in (B, C))
    G = B.shape[-2] if isinstance(B, Tensor) and B.dim() == nrows + 2 else 0
    if G < 1 or Dc % G:
        raise ValueError(f'B: {rows} + ([G,] {N}) with G a divisor of {Dc} expected, got {tuple(B.shape) if isinstance(B, Tensor) else B}')
    _like('B', B, u, rows + (G, N))
    _like('C', C, u, rows + (G, N))
    _like('state', state, u, (rows[0], Dc, N), _F32)
    _like('lengths', lengths, u, rows[:1], torch.int32)


def _norm_check(x, weight, residual, eps):
    _io('x', x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'x: [..., C] expected, got {tuple(x.shape)}')
    if x.shape[-1] > 1 << 30 or x.numel() // x.shape[-1] >= 1 << 31:
        raise ValueError(f'x: fewer than 2^31 rows of up to 2^30 columns expected, got {tuple(x.shape)}')
    _like('weight', weight, x, (x.shape[-1],), _F32)
    if weight is None:
        raise TypeError('weight: a tensor is wanted')
    if residual is not None:
        _like('residual', residual, x, x.shape, _F32 if isinstance(residual, Tensor) and residual.dtype == _F32 else x.dtype)
    if not eps >= 0.0:
        raise ValueError(f'{eps=}: not negative')


# ------------------------------------------------------------------------------------------------------------------ the operators
_ACT = {None: 0, 'linear': 0, 'silu': 1, 'swish': 1}


def short_conv(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = 'silu', state: Tensor | None = None,
               lengths: Tensor | None = None, return_state: bool = False):
    """Depthwise causal convolution: y[b, t, d] = act(bias[d] + sum_k weight[d, k] x[b, t - (K-1) + k, d]).

    x [B, L, D]; weight [D, K], K <= 8; activation 'silu' or None.  state [B, K-1, D] (x's type): the inputs in front of position 0, oldest first
    (None: zeros).  return_state: also the last K-1 inputs, the `state` of a call that goes on (from `state` itself where a sequence is shorter)."""
    out = _ops().short_conv(x, weight, bias, _ACT[activation], state, lengths, return_state) if activation in _ACT else None
    if out is None:
        _io('x', x)
        if x.dim() != 3:
            raise ValueError(f'x: [B, L, D] expected, got {tuple(x.shape)}')
        _conv_check(x, weight, bias, activation)
        _like('state', state, x, (x.shape[0], weight.shape[1] - 1, x.shape[2]))
        _like('lengths', lengths, x, (x.shape[0],), torch.int32)
        _refused('short_conv', x, weight, bias, state)
    return out


def short_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = 'silu',
                    state_out: Tensor | None = None) -> Tensor:
    """One position of `short_conv`: x [B, D], state [B, K-1, D] -> y [B, D].  The state moves on by one in place, or into state_out."""
    out = _ops().short_conv_step(x, state, weight, bias, _ACT[activation], state_out) if activation in _ACT else None
    if out is None:
        _no_grad_path('short_conv_step', x, state, weight, bias)
        _io('x', x)
        if x.dim() != 2:
            raise ValueError(f'x: [B, D] expected, got {tuple(x.shape)}')
        _conv_check(x, weight, bias, activation)
        _like('state', state, x, (x.shape[0], weight.shape[1] - 1, x.shape[1]))
        _state_check(state, state_out)
        _refused('short_conv_step', x, state, weight, bias, state_out)
    return out


def ssm_scan(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None, z: Tensor | None = None, dt_bias: Tensor | None = None,
             dt_softplus: bool = True, state: Tensor | None = None, lengths: Tensor | None = None, return_state: bool = False):
    """Selective state space scan.  With delta = softplus(dt + dt_bias) (dt_softplus=False: dt + dt_bias)

        h[b, t, d, n] = exp(delta A[d, n]) h[b, t-1, d, n] + delta u[b, t, d] B[b, t, g, n]
        y[b, t, d]    = (sum_n C[b, t, g, n] h[b, t, d, n] + D[d] u[b, t, d]) * silu(z[b, t, d])

    u, dt, z [B, L, D]; A [D, N], N <= 64 (negative for a stable scan); B, C [B, L, N] or [B, L, G, N]: channel d belongs to group d // (D / G);
    D, dt_bias [D].  Positions are walked in pieces side by side, each carried on by exp(A * its sum of delta): where that product leaves fp32's range (A * delta
    far above 0, a scan that grows) the result is not defined.  state [B, D, N]: h in front of position 0 (None: zeros).  return_state: also h at the end, the `state` of a call that goes on."""
    out = _ops().ssm_scan(u, dt, A, B, C, D, z, dt_bias, dt_softplus, state, lengths, return_state)
    if out is None:
        _ssm_check(u, dt, A, B, C, D, z, dt_bias, state, lengths, 2)
        for name, t in (('u', u), ('dt', dt), ('B', B), ('C', C), ('z', z)):
            if t is not None and t.shape[1] > 1 and t.stride(1) >= 1 << 22:
                raise lib.W2SError(f'{name}: positions lie {t.stride(1)} elements apart, 2^22 or more: pass a contiguous copy')
        _refused('ssm_scan', u, dt, A, B, C, D, z, dt_bias, state)
    return out


def ssm_step(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Tensor | None = None, z: Tensor | None = None,
             dt_bias: Tensor | None = None, dt_softplus: bool = True, state_out: Tensor | None = None) -> Tensor:
    """One position of `ssm_scan`: u, dt, z [B, D], B, C [B, N] or [B, G, N], state [B, D, N] fp32 -> y [B, D].  The state moves on in place, or
    into state_out."""
    out = _ops().ssm_step(u, dt, A, B, C, state, D, z, dt_bias, dt_softplus, state_out)
    if out is None:
        _no_grad_path('ssm_step', u, dt, A, B, C, state, D, z, dt_bias)
        _ssm_check(u, dt, A, B, C, D, z, dt_bias, state, None, 1)
        _state_check(state, state_out)
        _refused('ssm_step', u, dt, A, B, C, state, D, z, dt_bias, state_out)
    return out


def add_rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-5):
    """r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight over the last dimension; returns (y, r).  residual: x's type or fp32 (a residual stream
    in 32 bits), which is r's type; y has x's.  The sum is fp32 and y comes from it before r is rounded.  So is the mean of its squares: values beyond 1e19
    (with eps = 0 also a row below 1e-19) leave its range.  residual=None: r is x itself."""
    out = _ops().add_rms_norm(x, weight, residual, eps)
    if out is None:
        _norm_check(x, weight, residual, eps)
        _refused('add_rms_norm', x, weight, residual)
    return out


def add_rms_norm_8bit(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-5):
    """`add_rms_norm` with y in 8 bits: returns (q, scale, r), q float8_e4m3fn of x's shape, scale fp32 [...] with y ~ q * scale[..., None] -- the row-wise
    scaled operand of an 8-bit matrix product.  scale = max|y| / 448 over the row (1 for a row of zeros; NaN where the row holds one).  No backward."""
    out = _ops().add_rms_norm_8bit(x, weight, residual, eps)
    if out is None:
        _norm_check(x, weight, residual, eps)
        _no_grad_path('add_rms_norm_8bit', x, weight, residual)
        _refused('add_rms_norm_8bit', x, weight, residual)
    return out
