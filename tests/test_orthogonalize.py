# SPDX-License-Identifier: Apache-2.0
"""Argument checks of the orthogonalisation; nothing is launched and no GPU is needed."""
import ctypes

import pytest
import torch

from fastsafetensors_amd import _native, orthogonalize

F64, F32, F16, BF16, E4M3 = (_native.ELEM_TYPES[k] for k in ("F64", "F32", "F16", "BF16", "F8_E4M3"))
INVAL, RANGE = -10001, -10003
BASE = 0x10000000


def desc(dst=BASE, src=2 * BASE, rows=100, cols=300, pitch=None, strides=None, type=BF16):
    return _native.FstxOrthogonalizeDesc(dst, src, rows, cols, cols if pitch is None else pitch, *(strides or (cols, 1)), type, 0)


FIVE = (ctypes.c_float * 15)(*(3.4445, -4.775, 2.0315) * 5)


def need(*descs):
    return _native.lib().fstx_orthogonalize_workspace((_native.FstxOrthogonalizeDesc * len(descs))(*descs), len(descs), FIVE, 5)


def size(p, q):
    return (3 * p * q + 2 * p * p) * 4 + 8192  # X, two X^T, A and B in two terms; partial sums of squares


def test_workspace_sizes():
    assert need() == 0 and need(desc(rows=0)) == 0 and need(desc(cols=0)) == 0
    # operands padded to 256 x 256, and at most one round of workgroups' partial sums (512 tiles of 256 x 128)
    for rows, cols, p, q in ((100, 300, 256, 512), (300, 100, 256, 512), (33, 33, 256, 256), (1000, 2500, 1024, 2560)):
        got = need(desc(rows=rows, cols=cols))
        assert size(p, q) <= got <= size(p, q) + 512 * 256 * 128 * 4
    # up to 32 rows: the Gram matrix in parts of 256 columns, at most 128 of them
    assert need(desc(rows=1, cols=1)) == 2 * 8192 and need(desc(rows=32, cols=1000)) == 5 * 8192
    assert need(desc(rows=1 << 20, cols=5, strides=(5, 1), src=1 << 40)) == 129 * 8192
    small = [desc(dst=BASE + (i << 20), src=2 * BASE + (i << 20)) for i in range(50)]
    assert 20 * size(256, 512) <= need(*small) < 21 * size(256, 512) + 512 * 256 * 128 * 4  # twenty at a time
    large = [desc(dst=(i + 1) << 36, src=(i + 100) << 36, rows=16384, cols=16384) for i in range(3)]
    assert size(16384, 16384) <= need(*large) < 2 * size(16384, 16384)   # one at a time


@pytest.mark.parametrize("bad,code", [
    (dict(type=F64), INVAL), (dict(type=E4M3), INVAL), (dict(dst=0), INVAL), (dict(src=0), INVAL), (dict(dst=BASE + 1), INVAL),
    (dict(src=2 * BASE + 1), INVAL), (dict(pitch=299), INVAL), (dict(rows=(1 << 20) + 1), RANGE), (dict(rows=70000, cols=70000), RANGE),
    (dict(strides=(1 << 40, 1)), RANGE),
])
def test_bad_descriptors_are_refused(bad, code):
    assert need(desc(**bad)) == code


def test_overlaps():
    a = desc()
    assert need(a, desc(dst=3 * BASE)) > 0                       # the same source twice is fine
    assert need(a, desc(src=3 * BASE)) == INVAL                  # one destination twice
    assert need(a, desc(dst=2 * BASE)) == INVAL                  # a destination that another update reads
    assert need(desc(dst=BASE, src=BASE), desc(dst=3 * BASE)) > 0  # an update may be its own destination
    assert need(desc(dst=BASE, src=BASE + 2)) == INVAL           # but only exactly
    assert need(desc(dst=BASE, src=BASE, pitch=400)) == INVAL
    assert need(desc(dst=BASE, src=BASE, strides=(1, 100))) == INVAL


def test_steps_eps_and_workspace_are_checked():
    fn, arr, c = _native.lib().fstx_orthogonalize, (_native.FstxOrthogonalizeDesc * 1)(desc()), (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    n = _native.lib().fstx_orthogonalize_workspace(arr, 1, c, 1)
    assert n > 0
    for args in ((arr, 1, c, 0, 0.0, 0x1000, n), (arr, 1, c, 65, 0.0, 0x1000, n), (arr, 1, None, 1, 0.0, 0x1000, n),
                 (arr, 1, c, 1, -1.0, 0x1000, n), (arr, 1, c, 1, float("nan"), 0x1000, n), (arr, 1, c, 1, 0.0, None, n),
                 (arr, 1, c, 1, 0.0, 0x1010, n), (arr, 1, c, 1, 0.0, 0x1000, n - 1), (None, 1, c, 1, 0.0, 0x1000, n)):
        assert fn(*args, None) == INVAL
    assert fn(None, 0, c, 1, 0.0, None, 0, None) == 0


def test_python_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="GPU memory"):
        orthogonalize(torch.zeros(3, 4))
    for c in ([], [(1.0, 2.0)], [(1.0, 2.0, 3.0)] * 65):
        with pytest.raises(ValueError, match="triples"):
            orthogonalize([torch.zeros(3, 4)], coefficients=c)
    with pytest.raises(ValueError, match="finite"):
        orthogonalize([], coefficients=[(1.0, float("inf"), 0.0)])
    with pytest.raises(ValueError, match="finite"):
        orthogonalize([], eps=-1.0)
    with pytest.raises(ValueError, match="outs for"):
        orthogonalize([torch.zeros(3, 4)], outs=[])
    assert orthogonalize([]) == []
