"""The state space mixer's operators at the shapes of mixer_paths.py -- many runs, many tiles, many workgroups, many rows a workgroup -- and the 8-bit norm at odd
widths, against the plain 64-bit statements, with the tolerances of test_mixer_ops_gpu.py (they count roundings and hold for any size)."""
import pytest
import torch

import wav2sleep_amd as W
from tests import mixer_paths as P
from tests import mixer_reference as R
from tests.test_mixer_ops_gpu import DTYPES, check_conv, check_norm, check_scan, rnd, scan_inputs, wide_view

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('shape', P.CONV, ids=str)
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_conv_windows_slide_from_run_to_run(dtype, shape):
    check_conv(dtype, *shape, ragged=True, strided=True, seed=13)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_conv_windows_without_ends(dtype):
    check_conv(dtype, 8, 1031, 1032, 4, silu=False, state=False, bias=False, seed=14)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('shape', P.SCAN_WIDE, ids=str)
def test_scan_wide_tiles_one_behind_the_other(dtype, shape):
    check_scan(scan_inputs(dtype, *shape, seed=51, ragged=True, strided=True))


@pytest.mark.parametrize('dtype', ['f32', 'f16'])
@pytest.mark.parametrize('shape', P.SCAN_MANY, ids=str)
def test_scan_more_workgroups_than_cus(dtype, shape):
    check_scan(scan_inputs(dtype, *shape, seed=52, ragged=True, strided=True, gate=shape[4] > 1 or dtype == 'f16'))


@pytest.mark.parametrize('strided', [False, True])
@pytest.mark.parametrize('rows,C,dtype', P.NORM)
def test_norm_several_rows_a_workgroup(rows, C, dtype, strided):
    for res in ('same', None) if dtype == 'f32' else ('same', 'f32'):
        check_norm(dtype, (rows,), C, res, strided=strided, seed=C)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('C', [9, 61, 130, 1021, 1999, 4095, 8191, 16383, 33001])
@pytest.mark.parametrize('res', ['same', 'f32', None])
@pytest.mark.parametrize('strided', [False, True])
def test_norm_8bit_odd_widths(dtype, C, res, strided):
    dt, rt = DTYPES[dtype], torch.float32 if res == 'f32' else DTYPES[dtype]
    x, w, r = (3 * rnd(1, 19, C)).to(dt), rnd(2, C), rnd(3, 19, C, dtype=rt) if res else None
    want, mag = (R.norm(x, w, r, mag=m) for m in (False, True))
    if strided:
        x, r = wide_view(x), wide_view(r, 5) if res else None
    q, scale, s = W.add_rms_norm_8bit(x, w, r)
    top = want['y'].abs().amax(-1)
    # y: a sum of C squares (C + 8 half steps), root and division, three products; the scale: y's error over 448 and the rounding of its own division
    slack = (C + 24) * R.U32 * mag['y'].amax(-1)
    assert ((scale.double() - top / 448).abs() <= 4 * R.U32 * top / 448 + slack / 448).all()
    # half a step of e4m3 is 2^-4 of the value, 2^-10 near zero; the value before rounding carries the norm's fp32 error, and so does the scale
    off = (q.double() * scale.double()[:, None] - want['y']).abs()
    tol = 2.0 ** -4 * want['y'].abs() + 2.0 ** -10 * scale.double()[:, None] + 2 * slack[:, None]
    assert (off <= tol).all(), float((off - tol).max())
    if res:
        R.close(s, want['r'], mag['r'], 1, 'r')
