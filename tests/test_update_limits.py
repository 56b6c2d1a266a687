# SPDX-License-Identifier: Apache-2.0
"""Workspaces and limits of the kernels that change weights; nothing is launched and no GPU is needed."""
import ctypes

import torch

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


def test_coefficients_reach_what_is_said_of_them():
    """Singular values relative to the Frobenius norm, on a grid of 2 * 10^6 over six decades (steps of 7e-6 of a value,
    which slopes of up to 6000 turn into 4e-2 of it where a value is small, and into nothing that matters where it has converged)."""
    from fastsafetensors_amd.updates import DEFAULT_COEFFICIENTS, POLAR_COEFFICIENTS

    s = torch.logspace(-6, 0, 2_000_001, dtype=torch.float64)

    def outcome(coefficients):
        x = s
        for a, b, c in coefficients:
            x = a * x + b * x**3 + c * x**5
            assert x.max() < 1.21  # and iterates stay below 2
        return x

    five, polar = outcome(DEFAULT_COEFFICIENTS), outcome(POLAR_COEFFICIENTS)
    assert five[s >= 1.5e-3].min() >= 0.679 and abs(five[s <= 1e-3].max().item() - 0.47) < 0.01
    assert ((polar - 1).abs()[s >= 5e-4] < 3e-4).all() and ((polar - 1).abs()[s >= 7e-4] < 1e-6).all()
    assert abs(five[0].item() / 1e-6 - 484.9) < 0.5 and abs(polar[0].item() / 1e-6 - 5993) < 5  # a^5, times 1.875^4; cubic terms are below 1e-4 of it


def test_overlaps_are_those_of_the_bytes():
    """Pairs of blocks, small enough to list their bytes: what overlaps is refused, and what does not is taken where both have
    rows equally far apart or one is a single row (blocks of different pitches whose spans touch are not told apart)."""
    import random

    rng, base, fn = random.Random(5), 1 << 20, _native.lib().fstx_merge_low_rank_workspace
    told = 0
    for _ in range(20000):
        blocks, descs = [], []
        pitch = rng.randint(1, 9)
        for i in range(2):
            rows, own = rng.randint(1, 5), pitch if rng.random() < 0.7 else rng.randint(1, 9)
            cols = rng.randint(1, own if rows > 1 else 9)
            at = rng.randint(0, 40)
            blocks.append((at, rows, cols, own))
            descs.append(_native.FstxLowRankDesc(base + 2 * at, (2 + i) << 30, None, None, None, rows, cols, 0, own, cols, 0, 0, 0, 0, 1.0,
                                                 BF16, BF16, BF16, 0, 0))
        bytes_ = [{at + r * own + c for r in range(rows) for c in range(cols)} for at, rows, cols, own in blocks]
        got = fn((_native.FstxLowRankDesc * 2)(*descs), 2)
        (_, r0, c0, p0), (_, r1, c1, p1) = blocks
        if bytes_[0] & bytes_[1]:
            assert got == -10001, blocks
        elif p0 == p1 or r0 == r1 == 1 or (r0 == 1 and c0 <= p1) or (r1 == 1 and c1 <= p0):
            assert got == 0, blocks
            told += 1
    assert told > 5000
