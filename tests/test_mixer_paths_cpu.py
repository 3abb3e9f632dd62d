"""CPU-only: the shapes of mixer_paths.py take the paths that they stand for, as the sizes of the scratch memory that a call asks for tell."""
import ctypes
import os

import pytest

from tests import mixer_paths as P
from wav2sleep_amd import lib


@pytest.fixture(scope='module')
def dll():
    if not os.path.exists(lib.LIB_PATH):
        lib.build()
    return lib.load()


@pytest.mark.parametrize('shape', P.CONV, ids=str)
def test_a_thread_of_the_convolution_takes_several_runs(dll, shape):
    B, L, D, K = shape
    a = lib.ShortConvArgs(x=4096, w=4096, B=B, L=L, D=D, K=K, sx_b=L * D, sx_l=D)
    shares = dll.w2s_short_conv_part(ctypes.byref(a)) // (B * (K + 1) * D)   # the backward's workgroups along a sequence
    groups = -(-D // 4) if D >= 4 else D   # of channels
    lanes = 1
    while lanes < min(groups, 64):
        lanes *= 2
    one = -(-(-(-L // 4)) // (256 // lanes))   # ... with runs of four positions, one a thread
    assert shares < one
    assert B * -(-groups // lanes) * one > 2048   # so many workgroups that the forward takes several runs too


def scan(B, L, D, N, G):
    return lib.SsmArgs(A=4096, B=B, L=L, D=D, N=N, G=G, su_l=D, sdt_l=D, sB_l=N * G, sC_l=N * G)


def plan(dll, shape):
    """(tile of the backward, segments in the forward?, workgroups)"""
    B, L, D, N, G = shape
    a = ctypes.byref(scan(*shape))
    NP = 8 if N <= 8 else 16 if N <= 16 else 32 if N <= 32 else 64
    return dll.w2s_ssm_ckpt(a) // (B * D * NP), dll.w2s_ssm_ws(a, 0) > 0, B * G * -(-(D // G) // 16)


@pytest.mark.parametrize('shape', P.SCAN_WIDE, ids=str)
def test_wide_tiles_one_behind_the_other(dll, shape):
    marks, cut, blocks = plan(dll, shape)
    assert not cut and 128 < blocks <= 256 and marks == -(-shape[1] // 64) and marks > 8


@pytest.mark.parametrize('shape', P.SCAN_MANY, ids=str)
def test_narrow_tiles_of_more_workgroups_than_cus(dll, shape):
    marks, cut, blocks = plan(dll, shape)
    tile = 64 if 16 < shape[3] <= 32 else 32
    assert not cut and blocks > 256 and marks == -(-shape[1] // tile) and marks > 2


@pytest.mark.parametrize('rows,C,dtype', P.NORM)
def test_a_workgroup_of_the_norm_takes_several_rows(dll, rows, C, dtype):
    d = dict(f32=0, bf16=1, f16=2)[dtype]
    a = lib.AddNormArgs(x=4096, w=4096, rows=rows, C=C, ldx=C, dtype=d, rdtype=d)
    units = -(-C // (4 if d == 0 else 8))
    together = 16 if units <= 16 else 8 if units <= 32 else 4 if units <= 128 else 1   # rows a workgroup has side by side
    assert rows > together * dll.w2s_add_norm_part(ctypes.byref(a)) // C
