# SPDX-License-Identifier: Apache-2.0
"""Merges that run out of memory change nothing."""
import pytest
import torch

from fastsafetensors_amd import DType, LowRankUpdate, SafeTensorsFileLoader, SingleGroup, merge_low_rank, updates
from fastsafetensors_amd.checkpoints import TensorSpec, write_checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


@pytest.mark.parametrize("fails", [1, 2, 3])
def test_a_merge_cut_into_several_calls_changes_all_or_nothing(dev, monkeypatch, fails):
    g = torch.Generator().manual_seed(1)
    host = [tuple(torch.randn(*s, generator=g) for s in ((300, 500), (300, 64), (64, 500))) for _ in range(4)]
    items = [LowRankUpdate(*(t.to(dev) for t in h)) for h in host]
    monkeypatch.setattr(updates, "_WORKSPACE_BYTES", 1 << 19)  # each needs (512 + 512) * 64 * 6 bytes: four calls
    empty, asked = torch.empty, []

    def scarce(*args, **kw):
        asked.append(args)
        if len(asked) == fails:
            raise torch.OutOfMemoryError("no memory left")
        return empty(*args, **kw)

    monkeypatch.setattr(torch, "empty", scarce)
    try:
        merge_low_rank(items)
    except torch.OutOfMemoryError:
        for u, (w, _, _) in zip(items, host):
            assert torch.equal(u.weight.cpu(), w)
    else:
        for u, (w, up, down) in zip(items, host):
            want = w.double() + up.double() @ down.double()
            # 64 sums of products of about 1 (six per k) in 32 bits, and the weight added
            assert (u.weight.cpu().double() - want).abs().max() < 64 * 6 * 16 * 2.0**-24


def load(path):
    loader = SafeTensorsFileLoader(SingleGroup(), "cuda:0", max_threads=4)
    loader.add_filenames({0: [str(path)]})
    return loader, loader.copy_files_to_device()


def polar(d):
    """The nine steps of POLAR_COEFFICIENTS in 64 bits: singular values below 0.0005 of the norm, of which a square matrix has a few, do not reach 1."""
    x = d / (d.norm() + 1e-7)
    x = x.t().contiguous() if x.shape[0] > x.shape[1] else x
    for a, b, c in updates.POLAR_COEFFICIENTS:
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * s @ s) @ x
    return x.t() if d.shape[0] > d.shape[1] else x


def test_checkpoints_are_merged_all_or_nothing(dev, tmp_path, monkeypatch):
    """Vectors and matrices; whichever of the merge's allocations fails, nothing has changed."""
    specs = [TensorSpec("a.norm", DType.BF16, (64,)), TensorSpec("b.weight", DType.BF16, (300, 200)), TensorSpec("c.weight", DType.BF16, (2048, 2048))]
    for i in range(3):
        write_checkpoint(str(tmp_path / f"{i}.safetensors"), specs, i)
    loaded = [load(tmp_path / f"{i}.safetensors") for i in range(3)]
    bufs, others = loaded[0][1], [b for _, b in loaded[1:]]
    before = {s.name: bufs.get_tensor(s.name).clone() for s in specs}
    empty, asked, fails = torch.empty, [], 0

    def scarce(*args, **kw):
        asked.append(args)
        if len(asked) == fails:
            raise torch.OutOfMemoryError("no memory left")
        return empty(*args, **kw)

    while True:
        fails += 1
        asked.clear()
        with monkeypatch.context() as patch:
            patch.setattr(torch, "empty", scarce)
            try:
                names = bufs.merge_checkpoints(others)
            except torch.OutOfMemoryError:
                names = None
        if names is not None:
            break
        for name, w in before.items():
            assert torch.equal(bufs.get_tensor(name), w), (fails, name)
    assert fails > 1 and sorted(names) == sorted(before)
    for name, w in before.items():
        tuned = [o.get_tensor(name).double() for o in others]
        d = sum(t - w.double() for t in tuned)
        if w.dim() == 1:
            want = w.double() + d / 2
        else:
            o = polar(d)
            want = w.double() + (d * o).sum() / min(d.shape) * o
        # half a step of bf16 (of the norm; independent roundings come to 0.43 of that); the iteration itself rounds by
        # 2^-22 times 6000, the growth of the smallest directions: 1.4e-3 in these few, 2^-18 elsewhere
        assert (bufs.get_tensor(name).double() - want).norm() <= want.norm() * (torch.finfo(torch.bfloat16).eps / 2), name
    for loader, b in loaded:
        b.close()
        loader.close()
