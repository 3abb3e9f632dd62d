"""`SequenceSSM`: a causal state space mixer over epochs, in the place of `SequenceCNN` (reference models/wav2sleep.py:349-390, which mixes with dilated
convolutions over a fixed reach).  A layer is pre-norm residual: r += x; n = RMS norm of r; u, z = projections of n; u = short causal convolution of u;
(dt, B, C) = projections of u; x = projection of the selective scan of u, gated by z (mixer_ops.py).  Epoch t sees epochs <= t, whatever their number, and a
stream is mixed one epoch at a time: `step` costs the same for the first epoch and for the thousandth, where a causal SequenceCNN runs over its reach again.

    mixer = SequenceSSM(128, num_layers=2)
    model = Wav2Sleep(encoders, epoch_mixer, mixer, num_classes=4)      # trains through SleepModule / GenericTrainStep like any other configuration
    y, state = mixer.prompt(x_BSF)                                      # streaming: the night so far (or state = mixer.init_state(batch)), ...
    y = mixer.step(x_BF, state)                                         # ... then features of the newest epoch in, mixed features out

fp32, like the rest of the path around it.  There is no CPU path (lib.W2SError)."""
from __future__ import annotations

import math

import torch
from torch import Tensor, nn

from . import mixer_ops


class SSMLayer(nn.Module):
    """Parameters of one layer; `SequenceSSM` and generic.py's walker run it."""

    def __init__(self, feature_dim: int, inner_dim: int, state_dim: int, kernel_size: int, dt_rank: int):
        super().__init__()
        self.norm_weight = nn.Parameter(torch.ones(feature_dim))
        self.in_proj = nn.Linear(feature_dim, inner_dim, bias=False)
        self.gate_proj = nn.Linear(feature_dim, inner_dim, bias=False)
        bound = 1.0 / math.sqrt(kernel_size)
        self.conv_weight = nn.Parameter(torch.empty(inner_dim, kernel_size).uniform_(-bound, bound))
        self.conv_bias = nn.Parameter(torch.zeros(inner_dim))
        self.x_proj = nn.Linear(inner_dim, dt_rank + 2 * state_dim, bias=False)
        self.dt_proj = nn.Linear(dt_rank, inner_dim, bias=False)
        first = torch.exp(torch.rand(inner_dim) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))   # time steps of 0.001 ... 0.1 to begin with
        self.dt_bias = nn.Parameter(first + torch.log(-torch.expm1(-first)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, state_dim + 1, dtype=torch.float32)).repeat(inner_dim, 1))   # A = -exp(A_log)
        self.D = nn.Parameter(torch.ones(inner_dim))
        self.out_proj = nn.Linear(inner_dim, feature_dim, bias=False)


class SequenceSSM(nn.Module):
    causal = True
    compiled_with: dict | None = None

    def __init__(self, feature_dim: int = 128, dropout: float = 0.0, num_layers: int = 2, expand: int = 2, state_dim: int = 16, kernel_size: int = 4, dt_rank: int = 16,
                 norm_eps: float = 1e-5) -> None:
        super().__init__()
        if feature_dim % 16 or dt_rank % 16 or dt_rank < 16 or state_dim % 8 or not 8 <= state_dim <= 64 or not 1 <= kernel_size <= 8:
            raise ValueError(f'SequenceSSM: multiples of 16 for {feature_dim=} and {dt_rank=}, {state_dim=} in 8, 16, ... 64, {kernel_size=} in 1 ... 8')
        self.feature_dim, self.dropout_p, self.num_layers, self.expand = feature_dim, dropout, num_layers, expand
        self.state_dim, self.kernel_size, self.dt_rank, self.norm_eps = state_dim, kernel_size, dt_rank, norm_eps
        self.inner_dim = expand * feature_dim
        self.layers = nn.ModuleList([SSMLayer(feature_dim, self.inner_dim, state_dim, kernel_size, dt_rank) for _ in range(num_layers)])
        self.norm_weight = nn.Parameter(torch.ones(feature_dim))

    def fused_ok(self) -> bool:
        """not part of the production family's fused step: models with it run on the generic path"""
        return False

    def compile(self, *args, **kwargs):
        self.compiled_with = dict(args=args, **kwargs)   # (hand-written launches: there is nothing to compile)

    def config_dict(self) -> dict:
        return {'_target_': 'wav2sleep_amd.SequenceSSM', 'feature_dim': self.feature_dim, 'dropout': self.dropout_p, 'num_layers': self.num_layers, 'expand': self.expand,
                'state_dim': self.state_dim, 'kernel_size': self.kernel_size, 'dt_rank': self.dt_rank, 'norm_eps': self.norm_eps}

    @torch.no_grad()
    def forward(self, x_BSF: Tensor) -> Tensor:
        """[B, S, F] -> [B, S, F] (inference; training goes through Wav2Sleep.forward)."""
        from .wav2sleep import _gen
        gen = _gen(self)
        mixer_ops.no_forward_mode('SequenceSSM', x_BSF, *self.parameters())
        mixer_ops.no_trace('SequenceSSM')
        with torch.cuda.device(self.norm_weight.device):
            return gen.sequence_ssm(self, x_BSF)

    def init_state(self, batch: int) -> list:
        """per layer: (the convolution's last inputs, the scan's state) in front of the first epoch"""
        dev = self.norm_weight.device
        return [(torch.zeros(batch, self.kernel_size - 1, self.inner_dim, device=dev), torch.zeros(batch, self.inner_dim, self.state_dim, device=dev)) for _ in self.layers]

    def _mix(self, x: Tensor, state: list, conv, scan) -> Tensor:
        """rows x [R, F] through the layers; conv(k, u, state) and scan(k, u, dt, A, B, C, z, state) are layer k's operators"""
        from .wav2sleep import _gen
        gen = _gen(self)
        gen.training = False
        r, N = self.dt_rank, self.state_dim
        with torch.cuda.device(self.norm_weight.device):
            x, res = x.float().contiguous(), None
            for k, (layer, (conv_state, h)) in enumerate(zip(self.layers, state)):
                n, res = mixer_ops.add_rms_norm(x, layer.norm_weight, res, self.norm_eps)
                u = conv(k, gen.linear(n, layer.in_proj.weight, None), conv_state)
                dbc = gen.linear(u, layer.x_proj.weight, None)
                dt = gen.linear(dbc[:, :r].contiguous(), layer.dt_proj.weight, None)
                y = scan(k, u, dt, -torch.exp(layer.A_log), dbc[:, r:r + N], dbc[:, r + N:], gen.linear(n, layer.gate_proj.weight, None), h)
                x = gen.linear(y, layer.out_proj.weight, None)
            return mixer_ops.add_rms_norm(x, self.norm_weight, res, self.norm_eps)[0]

    def _state_check(self, state: list, batch: int, moves: bool):
        """in front of the first layer, so that a refused step has moved no layer's state; moves: the state is written to, so it has to lie as it is written"""
        if len(state) != len(self.layers):
            raise ValueError(f'the state of {len(self.layers)} layers expected, got {len(state)}')
        want = ((batch, self.kernel_size - 1, self.inner_dim), (batch, self.inner_dim, self.state_dim))
        for k, pair in enumerate(state):
            if len(pair) != 2 or any(tuple(t.shape) != w or t.dtype != torch.float32 for t, w in zip(pair, want)):
                raise ValueError(f'layer {k}: a state of fp32 tensors {want[0]} and {want[1]} expected, got {[(tuple(t.shape), t.dtype) for t in pair]}')
            if moves and not all(t.is_contiguous() and t.device == self.norm_weight.device and not t.requires_grad for t in pair):
                raise ValueError(f'layer {k}: a step writes its state in place: contiguous tensors on {self.norm_weight.device} that want no gradient expected')

    @torch.no_grad()
    def prompt(self, x_BSF: Tensor, lengths: Tensor | None = None, state: list | None = None):
        """The epochs of a night so far, [B, S, F] -> (mixed features [B, S, F], state behind them for `step` or another `prompt`).  lengths (int32 [B], on the
        device): how many of the S epochs each sequence has; features behind them are of no meaning.  state: what stands in front (None: nothing)."""
        if x_BSF.dim() != 3 or x_BSF.shape[2] != self.feature_dim or x_BSF.shape[0] < 1 or x_BSF.shape[1] < 1:
            raise ValueError(f'[B, S, {self.feature_dim}] with one epoch at least expected, got {tuple(x_BSF.shape)}')
        B, S, _ = x_BSF.shape
        state = self.init_state(B) if state is None else state
        self._state_check(state, B, False)
        behind = [[None, None] for _ in self.layers]
        seq = lambda t: t.unflatten(0, (B, S))   # noqa: E731

        def conv(k, u, st):
            p = self.layers[k]
            y, behind[k][0] = mixer_ops.short_conv(seq(u), p.conv_weight, p.conv_bias, state=st, lengths=lengths, return_state=True)
            return y.flatten(0, 1)

        def scan(k, u, dt, A, Bm, Cm, z, h):
            p = self.layers[k]
            y, behind[k][1] = mixer_ops.ssm_scan(seq(u), seq(dt), A, seq(Bm), seq(Cm), D=p.D, z=seq(z), dt_bias=p.dt_bias, state=h, lengths=lengths, return_state=True)
            return y.flatten(0, 1)
        y = self._mix(x_BSF.reshape(B * S, -1), state, conv, scan)
        return y.view(B, S, -1), [tuple(s) for s in behind]

    @torch.no_grad()
    def step(self, x_BF: Tensor, state: list) -> Tensor:
        """The newest epoch's features [B, F] -> mixed features [B, F]; `state` (init_state, or what prompt returned) moves on in place."""
        if x_BF.dim() != 2 or x_BF.shape[1] != self.feature_dim:
            raise ValueError(f'[B, {self.feature_dim}] expected, got {tuple(x_BF.shape)}')
        self._state_check(state, x_BF.shape[0], True)

        def conv(k, u, st):
            p = self.layers[k]
            return mixer_ops.short_conv_step(u, st, p.conv_weight, p.conv_bias)

        def scan(k, u, dt, A, Bm, Cm, z, h):
            p = self.layers[k]
            return mixer_ops.ssm_step(u, dt, A, Bm, Cm, h, D=p.D, z=z, dt_bias=p.dt_bias)
        return self._mix(x_BF, state, conv, scan)
