"""`SequenceSSM`: a causal state space mixer over epochs, in the place of `SequenceCNN` (reference models/wav2sleep.py:349-390, which mixes with dilated
convolutions over a fixed reach).  A layer is pre-norm residual: r += x; n = RMS norm of r; u, z = projections of n; u = short causal convolution of u;
(dt, B, C) = projections of u; x = projection of the selective scan of u, gated by z (mixer_ops.py).  Epoch t sees epochs <= t, whatever their number, and a
stream is mixed one epoch at a time: `step` costs the same for the first epoch and for the thousandth, where a causal SequenceCNN runs over its reach again.

    mixer = SequenceSSM(128, num_layers=2)
    model = Wav2Sleep(encoders, epoch_mixer, mixer, num_classes=4)      # trains through SleepModule / GenericTrainStep like any other configuration
    state = mixer.init_state(batch)                                     # streaming: features of the newest epoch in, mixed features out
    y = mixer.step(x_BF, state)

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
        with torch.cuda.device(self.norm_weight.device):
            return gen.sequence_ssm(self, x_BSF)

    def init_state(self, batch: int) -> list:
        """per layer: (the convolution's last inputs, the scan's state) in front of the first epoch"""
        dev = self.norm_weight.device
        return [(torch.zeros(batch, self.kernel_size - 1, self.inner_dim, device=dev), torch.zeros(batch, self.inner_dim, self.state_dim, device=dev)) for _ in self.layers]

    @torch.no_grad()
    def step(self, x_BF: Tensor, state: list) -> Tensor:
        """The newest epoch's features [B, F] -> mixed features [B, F]; `state` (init_state, or an earlier step's) moves on in place."""
        from .wav2sleep import _gen
        if x_BF.dim() != 2 or x_BF.shape[1] != self.feature_dim:
            raise ValueError(f'[B, {self.feature_dim}] expected, got {tuple(x_BF.shape)}')
        if len(state) != len(self.layers):
            raise ValueError(f'the state of {len(self.layers)} layers expected, got {len(state)}')
        gen = _gen(self)
        gen.training = False
        r, N, rank = self.dt_rank, self.state_dim, self.dt_rank
        with torch.cuda.device(self.norm_weight.device):
            x, res = x_BF.float().contiguous(), None
            for layer, (conv_state, h) in zip(self.layers, state):
                n, res = mixer_ops.add_rms_norm(x, layer.norm_weight, res, self.norm_eps)
                u = mixer_ops.short_conv_step(gen.linear(n, layer.in_proj.weight, None), conv_state, layer.conv_weight, layer.conv_bias)
                dbc = gen.linear(u, layer.x_proj.weight, None)
                dt = gen.linear(dbc[:, :rank].contiguous(), layer.dt_proj.weight, None)
                y = mixer_ops.ssm_step(u, dt, -torch.exp(layer.A_log), dbc[:, r:r + N], dbc[:, r + N:], h, D=layer.D, z=gen.linear(n, layer.gate_proj.weight, None),
                                       dt_bias=layer.dt_bias)
                x = gen.linear(y, layer.out_proj.weight, None)
            return mixer_ops.add_rms_norm(x, self.norm_weight, res, self.norm_eps)[0]
