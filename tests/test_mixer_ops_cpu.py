"""CPU-only checks of the state space mixer's operators: descriptor layouts, refusals of the C entry points and of the public functions."""
import ctypes
import os
import subprocess

import pytest
import torch

import wav2sleep_amd as W
from wav2sleep_amd import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def dll():
    if not os.path.exists(lib.LIB_PATH):
        lib.build()
    return lib.load()


def test_descriptors_match_the_header(tmp_path):
    pairs = [('w2s_short_conv_args', lib.ShortConvArgs), ('w2s_ssm_args', lib.SsmArgs), ('w2s_add_norm_args', lib.AddNormArgs)]
    prints, want = [], []
    for c, s in pairs:
        prints.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(s))
        for f, _ in s._fields_:
            prints.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(s, f).offset)
    src = tmp_path / 't.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "w2s.h"\nint main(void){' + '\n'.join(prints) + 'return 0;}\n')
    exe = tmp_path / 't'
    subprocess.check_call(['gcc', '-std=c99', '-Wall', '-Werror', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)])
    assert [int(v) for v in subprocess.check_output([str(exe)]).split()] == want


def test_c_entries_refuse_bad_descriptors(dll):
    r = ctypes.byref
    for name in ('w2s_short_conv_fwd', 'w2s_short_conv_bwd', 'w2s_short_conv_step', 'w2s_ssm_scan_fwd', 'w2s_ssm_scan_bwd', 'w2s_ssm_step', 'w2s_add_norm_fwd', 'w2s_add_norm_bwd'):
        assert getattr(dll, name)(None, None) == -1, name
    for name, more in (('w2s_short_conv_part', ()), ('w2s_ssm_ckpt', ()), ('w2s_ssm_ws', (1,)), ('w2s_add_norm_part', ())):
        assert getattr(dll, name)(None, *more) == -1, name

    def conv(**kw):
        a = lib.ShortConvArgs(x=4096, w=4096, y=4096, gx=4096, state=4096, state_out=4096, B=1, L=8, D=16, K=4, sx_b=128, sx_l=16)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for kw in (dict(K=0), dict(K=9), dict(D=0), dict(B=-1), dict(L=-1), dict(dtype=3), dict(act=2), dict(w=None), dict(x=None), dict(y=None)):
        assert dll.w2s_short_conv_fwd(r(conv(**kw)), None) == -1, kw
    assert dll.w2s_short_conv_fwd(r(conv(B=0)), None) == 0 and dll.w2s_short_conv_fwd(r(conv(L=0, state_out=None)), None) == 0
    for kw in (dict(gx=None), dict(gw=4096), dict(K=9), dict(B=0, gw=4096, part=4096)):
        assert dll.w2s_short_conv_bwd(r(conv(**kw)), None) == -1, kw
    for kw in (dict(state=None), dict(state_out=None), dict(x=None), dict(K=9)):
        assert dll.w2s_short_conv_step(r(conv(**kw)), None) == -1, kw
    assert dll.w2s_short_conv_fwd(r(conv(B=0x7fffffff, L=0x7fffffff, D=4096)), None) == -1   # more workgroups than a launch takes

    def ssm(**kw):
        a = lib.SsmArgs(u=4096, dt=4096, Bm=4096, Cm=4096, A=4096, y=4096, h_out=4096, gu=4096, gdt=4096, gB=4096, gC=4096, gA=4096, ws=4096, B=1, L=8, D=16, N=16, G=1)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for kw in (dict(N=0), dict(N=65), dict(G=0), dict(G=3), dict(D=0), dict(dtype=-1), dict(B=-1), dict(A=None), dict(u=None), dict(dt=None), dict(Bm=None), dict(Cm=None), dict(y=None)):
        assert dll.w2s_ssm_scan_fwd(r(ssm(**kw)), None) == -1, kw
    assert dll.w2s_ssm_scan_fwd(r(ssm(B=0)), None) == 0
    for kw in (dict(gA=None), dict(ws=None), dict(gu=None), dict(gdt=None), dict(gB=None), dict(gC=None), dict(z=4096), dict(N=65)):
        assert dll.w2s_ssm_scan_bwd(r(ssm(**kw)), None) == -1, kw
    for kw in (dict(h_out=None), dict(u=None), dict(N=65), dict(G=3)):
        assert dll.w2s_ssm_step(r(ssm(**kw)), None) == -1, kw

    def norm(**kw):
        a = lib.AddNormArgs(x=4096, w=4096, y=4096, rstd=4096, rows=2, C=16, ldx=16)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for kw in (dict(C=0), dict(rows=-1), dict(dtype=3), dict(dtype=1, rdtype=2), dict(rdtype=1), dict(x=None), dict(y=None), dict(w=None), dict(res=4096), dict(r=4096), dict(fp8=1)):
        assert dll.w2s_add_norm_fwd(r(norm(**kw)), None) == -1, kw
    assert dll.w2s_add_norm_fwd(r(norm(rows=0)), None) == 0
    for kw in (dict(fp8=1), dict(gw=4096), dict(x=None), dict(rstd=None)):
        assert dll.w2s_add_norm_bwd(r(norm(**kw)), None) == -1, kw


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 4, 8), torch.zeros(8, 4)
    for call in (lambda: W.short_conv(x, w), lambda: W.short_conv_step(x[:, 0], torch.zeros(2, 3, 8), w),
                 lambda: W.ssm_scan(x, x, w, torch.zeros(2, 4, 4), torch.zeros(2, 4, 4)),
                 lambda: W.ssm_step(x[:, 0], x[:, 0], w, torch.zeros(2, 4), torch.zeros(2, 4), torch.zeros(2, 8, 4)),
                 lambda: W.add_rms_norm(x, torch.ones(8)), lambda: W.add_rms_norm_8bit(x, torch.ones(8), x)):
        with pytest.raises(W.lib.W2SError):
            call()
    with pytest.raises(TypeError):
        W.add_rms_norm([1.0], torch.ones(1))
