# SPDX-License-Identifier: Apache-2.0
"""Argument checks of the low-rank merge; nothing is launched and no GPU is needed."""
import ctypes
import os
import re

import pytest
import torch

from conftest import ROOT
from fastsafetensors_amd import LowRankUpdate, _native, merge_low_rank

F32, F16, BF16, E4M3 = (_native.ELEM_TYPES[k] for k in ("F32", "F16", "BF16", "F8_E4M3"))
SIZE = {F32: 4, F16: 2, BF16: 2, E4M3: 1}
INVAL, RANGE = -10001, -10003


def desc(dst=0x1000000, src=None, rows=100, cols=60, rank=8, type=BF16, pitch=None, src_pitch=None, up=0x8000000, down=0x9000000,
         ftype=BF16, ws=None, n_ws=0, scale=1.0, up_strides=None, down_strides=None):
    pitch = cols if pitch is None else pitch
    us, ds = up_strides or (rank, 1), down_strides or (cols, 1)
    return _native.FstxLowRankDesc(dst, dst if src is None else src, up, down, ws, rows, cols, rank, pitch,
                                   pitch if src_pitch is None else src_pitch, *us, *ds, scale, type, ftype, ftype, n_ws, 0)


def need(*descs):
    arr = (_native.FstxLowRankDesc * len(descs))(*descs)
    return _native.lib().fstx_merge_low_rank_workspace(arr, len(descs))


def test_header_and_binding_list_the_same_functions_and_layouts(tmp_path):
    text = open(os.path.join(ROOT, "include", "fstx_update.h")).read()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(fstx_[a-z0-9_]+)\s*\(", code))
    assert declared == set(_native.UPDATE_SYMBOLS)
    raw = ctypes.CDLL(_native.library_path())
    assert all(hasattr(raw, name) for name in declared)


def test_workspace_sizes():
    assert need() == 0
    assert need(desc(rows=0)) == need(desc(cols=0)) == need(desc(rank=0, up=None, down=None)) == 0
    assert need(desc()) == 0  # few tiles, a small rank: no packed factors
    # 100 x 60 at rank 64, padded to (256 + 256) rows of 64 k, 2 bytes, one term
    assert need(desc(rank=64)) == 512 * 64 * 2
    assert need(desc(rank=64, ftype=F32)) == 2 * 512 * 64 * 2
    assert need(desc(rank=64, ftype=F32, type=F32)) == 3 * 512 * 64 * 2
    assert need(desc(rank=33)) == 512 * 64 * 2
    assert need(desc(rank=64), desc(dst=0x2000000)) == 512 * (64 + 32) * 2
    far = 1 << 44
    assert need(desc(rows=1 << 15, cols=1 << 15, up=far, down=2 * far)) == (2 << 15) * 32 * 2


@pytest.mark.parametrize("bad", [
    dict(type=0), dict(type=5), dict(type=77), dict(ftype=E4M3), dict(ftype=0), dict(dst=0), dict(src=0x1000001), dict(dst=0x1000001),
    dict(up=None), dict(down=None), dict(up=0x8000001), dict(pitch=59), dict(src_pitch=59), dict(pitch=1 << 41),
    dict(ws=0x7000000, n_ws=1), dict(n_ws=1), dict(type=E4M3), dict(type=E4M3, ws=0x7000000, n_ws=7), dict(type=E4M3, ws=0x7000002, n_ws=1),
    dict(src=0x1000002), dict(src=0x1000000 + 100 * 60 * 2 - 2),       # a source the destination runs into
    dict(pitch=120, src_pitch=60), dict(src=0x1000000, pitch=60, src_pitch=120),
    dict(up=0x1000000), dict(down=0x1000000 + 2 * 5999), dict(up=0x1000000 - 2 * 799),  # factors inside the destination
])
def test_bad_descriptors_are_refused(bad):
    assert need(desc(**bad)) == INVAL
    arr = (_native.FstxLowRankDesc * 1)(desc(**bad))
    assert _native.lib().fstx_merge_low_rank(arr, 1, 0x100, 1 << 40, None) == INVAL  # before anything is launched


def test_sizes_out_of_range_are_refused():
    assert need(desc(rows=1 << 31)) == RANGE
    assert need(desc(cols=1 << 31, pitch=1 << 31)) == RANGE
    assert need(desc(rank=1 << 31)) == RANGE
    assert need(desc(up_strides=(1 << 31, 1))) == RANGE
    far = 1 << 44
    assert need(desc(rows=1 << 30, cols=1 << 20, pitch=1 << 20, up=far, down=2 * far)) == RANGE  # more tiles than a launch takes


def test_workspace_must_be_there_aligned_and_large_enough():
    arr = (_native.FstxLowRankDesc * 1)(desc(rank=64))
    fn, size = _native.lib().fstx_merge_low_rank, need(desc(rank=64))
    assert fn(arr, 1, None, size, None) == INVAL
    assert fn(arr, 1, 0x5000010, size, None) == INVAL
    assert fn(arr, 1, 0x5000000, size - 1, None) == INVAL
    assert fn(None, 1, None, 0, None) == INVAL
    assert fn(None, 0, None, 0, None) == 0


def test_overlaps_between_updates():
    a = desc()
    assert need(a, desc()) == INVAL                                     # the same weight twice
    assert need(a, desc(dst=0x1000000 + 60 * 2 * 50)) == INVAL          # rows in common
    assert need(a, desc(dst=0x3000000, src=0x1000000)) == INVAL         # one reads what the other writes
    assert need(a, desc(dst=0x3000000, up=0x1000000 + 64)) == INVAL
    assert need(a, desc(dst=0x1000000 + 100 * 60 * 2)) >= 0              # side by side
    # column blocks of one tensor with rows of 120
    left, right = desc(pitch=120), desc(dst=0x1000000 + 120, pitch=120)
    assert need(left, right) >= 0 and need(right, left) >= 0
    assert need(left, desc(dst=0x1000000 + 118, pitch=120)) == INVAL    # one column in common
    assert need(desc(dst=0x1000000 + 118, pitch=120), left) == INVAL
    assert need(right, desc(dst=0x1000000 + 240, pitch=120)) >= 0        # the next row's left block
    assert need(right, desc(dst=0x1000000 + 242, pitch=120)) == INVAL   # ... running into the row after it
    assert need(desc(dst=0x1000000, src=0x1000000 + 120, pitch=120)) >= 0  # out of place between two column blocks


def test_weight_scales_are_not_written_over():
    assert need(desc(type=E4M3, ws=0x7000000, n_ws=100)) >= 0
    assert need(desc(type=E4M3, ws=0x1000000 + 400, n_ws=1)) == INVAL
    assert need(desc(), desc(dst=0x3000000, type=E4M3, ws=0x1000000 + 100 * 60 * 2 - 4, n_ws=100)) == INVAL


def test_spans_beyond_memory_are_refused():
    assert need(desc(rows=1 << 20, cols=8, pitch=1 << 39)) == RANGE


def test_overlaps_among_thousands_of_updates():
    """Blocks of columns of one tensor, whole tensors and factors, in any order; one overlap anywhere is found."""
    import random

    descs = [desc(dst=(1 << 40) + i * 12000, up=(1 << 41) + i * 1600, down=(1 << 42) + i * 960) for i in range(6000)]
    descs += [desc(dst=(1 << 43) + i * 120, pitch=60 * 40, up=(1 << 41) + i * 1600, down=(1 << 42) + i * 960) for i in range(40)]
    random.Random(1).shuffle(descs)
    assert need(*descs) == 6040 * 512 * 32 * 2  # (too many tiles to go without packed factors)
    for bad in (desc(dst=(1 << 40) + 4000 * 12000 + 11998, up=1 << 20, down=1 << 21, rows=1), desc(dst=(1 << 43) + 118, pitch=60 * 40),
                desc(dst=(1 << 41) + 1600 * 3), desc(dst=1 << 44, src=(1 << 40) + 6000 * 12000 - 2)):
        assert need(*descs, bad) == INVAL and need(bad, *descs) == INVAL


def test_struct_layouts_are_the_headers(tmp_path):
    """Offsets and sizes of both descriptors as a C compiler lays them out."""
    import subprocess

    lines = []
    for struct, cls in (("fstx_low_rank_desc", _native.FstxLowRankDesc), ("fstx_orthogonalize_desc", _native.FstxOrthogonalizeDesc)):
        lines += [f'_Static_assert(offsetof({struct}, {name}) == {getattr(cls, name).offset}, "{name}");' for name, _ in cls._fields_]
        lines.append(f'_Static_assert(sizeof({struct}) == {ctypes.sizeof(cls)}, "{struct}");')
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include "fstx_update.h"\n' + "\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(source)], check=True)


def test_python_refuses_what_is_not_in_gpu_memory():
    w, u, d = torch.zeros(4, 6), torch.zeros(4, 2), torch.zeros(2, 6)
    with pytest.raises(ValueError, match="GPU memory"):
        merge_low_rank([LowRankUpdate(w, u, d)])
    with pytest.raises(TypeError, match="torch.Tensor"):
        merge_low_rank([LowRankUpdate(None, u, d)])
    assert merge_low_rank([]) == []
