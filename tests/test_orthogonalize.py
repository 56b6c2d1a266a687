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


def test_blocks_of_one_tensor_do_not_overlap():
    left, right = desc(pitch=600, src=BASE, strides=(600, 1)), desc(dst=BASE + 600, src=BASE + 600, pitch=600, strides=(600, 1))
    assert need(left, right) > 0 and need(right, left) > 0
    assert need(left, desc(dst=BASE + 598, src=3 * BASE, pitch=600)) == INVAL
    # an update stored by columns beside the columns that another result is stored in
    assert need(desc(dst=3 * BASE, src=BASE, strides=(1, 200)), desc(dst=BASE + 200, src=BASE + 200, rows=300, cols=100, pitch=200, strides=(200, 1))) > 0
    many = [desc(dst=(1 << 40) + i * 60000, src=(1 << 41) + i * 60000) for i in range(6000)]
    assert need(*many) > 0 and need(*many, desc(dst=(1 << 41) + 6000 * 60000 - 2, src=1 << 20)) == INVAL


def test_kinds_of_matrices_beyond_those_kept():
    """Thirty and more kinds (by the steps that run on shorter operands) in one call plan as each of them alone."""
    c = (ctypes.c_float * 192)(*[v for _ in range(64) for v in (1.05, 0.1, 0.01)])
    fn = _native.lib().fstx_orthogonalize_workspace
    descs = [desc(dst=(1 << 44) + (i << 36), src=(1 << 45) + (i << 36), rows=int(512 * 1.11**i), cols=int(512 * 1.11**i)) for i in range(46)]
    each = [fn((_native.FstxOrthogonalizeDesc * 1)(d), 1, c, 64) for d in descs]
    assert fn((_native.FstxOrthogonalizeDesc * 46)(*descs), 46, c, 64) == max(each)


def test_steps_eps_and_workspace_are_checked():
    fn, arr, c = _native.lib().fstx_orthogonalize, (_native.FstxOrthogonalizeDesc * 1)(desc()), (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    n = _native.lib().fstx_orthogonalize_workspace(arr, 1, c, 1)
    assert n > 0
    for args in ((arr, 1, c, 0, 0.0, 0x1000, n), (arr, 1, c, 65, 0.0, 0x1000, n), (arr, 1, None, 1, 0.0, 0x1000, n),
                 (arr, 1, c, 1, -1.0, 0x1000, n), (arr, 1, c, 1, float("nan"), 0x1000, n), (arr, 1, c, 1, float("inf"), 0x1000, n),
                 (arr, 1, (ctypes.c_float * 3)(1.0, float("nan"), 0.0), 1, 0.0, 0x1000, n), (arr, 1, c, 1, 0.0, None, n),
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
    with pytest.raises(ValueError, match="32-bit"):
        orthogonalize([], coefficients=[(1e39, 0.0, 0.0)])
    with pytest.raises(ValueError, match="outs for"):
        orthogonalize([torch.zeros(3, 4)], outs=[])
    assert orthogonalize([]) == []
