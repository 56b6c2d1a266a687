# SPDX-License-Identifier: Apache-2.0
"""Views whose memory does not hold their values are refused."""
import pytest
import torch

from fastsafetensors_amd import LowRankUpdate, merge_low_rank, orthogonalize

pytestmark = pytest.mark.gpu


def test_negated_views():
    dev = torch.device("cuda:0")
    make = torch.Generator().manual_seed(1)
    w, up, down, g = (torch.randn(*s, generator=make).to(dev) for s in ((40, 30), (40, 4), (4, 30), (40, 30)))

    def negated(t):
        view = torch.complex(torch.zeros_like(t), -t).conj().imag
        assert view.is_neg() and torch.equal(view, t)
        return view

    before = w.clone()
    for u in (LowRankUpdate(w, negated(up), down), LowRankUpdate(w, up, negated(down)), LowRankUpdate(negated(w), up, down),
              LowRankUpdate(w, up, down, out=negated(w)),
              LowRankUpdate(torch.zeros(40, 30, dtype=torch.float8_e4m3fn, device=dev), up, down, weight_scale=negated(torch.ones(1, device=dev)))):
        with pytest.raises(ValueError, match="resolve_neg"):
            merge_low_rank([u])
    assert torch.equal(w, before)
    for args in (dict(updates=negated(g)), dict(updates=[g], outs=[negated(g)])):
        with pytest.raises(ValueError, match="resolve_neg"):
            orthogonalize(**args)
    got = merge_low_rank([LowRankUpdate(negated(w).resolve_neg(), up, down)])[0]
    assert (got.double() - (before.double() + up.double() @ down.double())).abs().max() < 1e-5  # 4 sums of values of about 10 in 32 bits
