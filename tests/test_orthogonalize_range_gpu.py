# SPDX-License-Identifier: Apache-2.0
"""Iterates much larger than usual: singular values up to 2."""
import pytest
import torch

from fastsafetensors_amd import orthogonalize

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def iterate(x, coefficients, eps):
    x = x.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + eps)
    for a, b, c in coefficients:
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
    return x.t() if flip else x


@pytest.mark.parametrize("steps", [[(1.0, 0.5, 0.5)] * 2, [(1.9, 0.0, 0.0), (0.0, 0.0, 0.05)], [(2.0, 0.0, 0.0), (0.0, 1.0, 0.0)],
                                   [(1.0, 0.5, 0.5), (0.5, 0.0, 0.0), (1.0, 0.5, 0.5)], [(1.99, 0.0, 0.0), (-1.0, -2.0, -3.0)]])
def test_singular_values_up_to_two(dev, steps):
    """The polynomials of a single element, through the general path (more than 32 rows), the slim one and dense directions."""
    s = 1.0
    for a, b, c in steps:
        assert s <= 2.0
        s = a * s + b * s**3 + c * s**5
    for rows in (8, 40, 300):
        g = torch.zeros(rows, 300)
        g[5, 7] = 3.0
        got = orthogonalize(g.to(dev), coefficients=steps, eps=0.0).cpu()
        # one number: roundings of 2^-22 of X, A and B and of what their products leave out, in two or three steps with
        # slopes (s p' / p) of 5 at most: 2^-22 * 9 * (1 + 5 + 25)
        assert abs(got[5, 7].item() - s) <= abs(s) * 7e-5, (rows, got[5, 7].item(), s)
        assert got.count_nonzero() == 1
        row = torch.zeros(rows, 300)
        row[5] = torch.randn(300, generator=torch.Generator().manual_seed(rows))
        want = iterate(row, steps, 0.0)
        assert ((orthogonalize(row.to(dev), coefficients=steps, eps=0.0).cpu().double() - want).norm() <= want.norm() * 7e-5).all()
