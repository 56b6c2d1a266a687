# SPDX-License-Identifier: Apache-2.0
"""Merges that run out of memory change nothing."""
import pytest
import torch

from fastsafetensors_amd import LowRankUpdate, merge_low_rank, updates

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
