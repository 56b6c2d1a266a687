# SPDX-License-Identifier: Apache-2.0
"""Workspaces and limits of the kernels that change weights; nothing is launched and no GPU is needed."""
import ctypes

from fastsafetensors_amd import _native

F32, F16, BF16 = (_native.ELEM_TYPES[k] for k in ("F32", "F16", "BF16"))


def update(rows, cols, i=0, type=F32):
    return _native.FstxOrthogonalizeDesc((1 << 44) + (i << 34), (1 << 45) + (i << 34), rows, cols, cols, cols, 1, type, 0)


def need(steps, *descs):
    c = (ctypes.c_float * (3 * len(steps)))(*[v for s in steps for v in s])
    return _native.lib().fstx_orthogonalize_workspace((_native.FstxOrthogonalizeDesc * len(descs))(*descs), len(descs), c, len(steps))


def test_slim_matrices_and_many_steps_take_room_for_the_iterate():
    """Steps that let small directions grow by 2^13 at most are one run; between two runs X stands in 64 bits."""
    polar, quintic = (1.875, -1.25, 0.375), (3.4445, -4.775, 2.0315)
    squares = 5 * 8192  # the Gram matrix of [32, 1000] in four parts, and Q
    for steps, runs in (([quintic] * 5 + [polar] * 4, 1), ([polar] * 14, 1), ([polar] * 15, 2), ([quintic] * 7, 1), ([quintic] * 8, 2),
                        ([(1e30, 0.0, 0.0)], 1), ([(1e30, 0.0, 0.0), (1.0, 0.0, 0.0)], 2), ([(0.5, 0.1, 0.0)] * 64, 1), ([(-1.875, 1.0, 0.0)] * 15, 2)):
        assert need(steps, update(32, 1000)) == squares + (32 * 1000 * 8 if runs > 1 else 0), steps
        assert need(steps, update(1000, 32)) == squares + (32 * 1000 * 8 if runs > 1 else 0), steps
    # as many matrices at a time as 4 GiB hold: an iterate of [32, 2^20] takes 256 MiB
    one = need([polar] * 64, update(32, 1 << 20))
    assert one == 129 * 8192 + (32 << 23)
    assert need([polar] * 64, *[update(32, 1 << 20, i) for i in range(40)]) == (4 << 30) // one * one
