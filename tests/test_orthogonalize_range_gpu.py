# SPDX-License-Identifier: Apache-2.0
"""Iterates much smaller or larger than usual: updates far below eps, singular values up to 2."""
import pytest
import torch

from fastsafetensors_amd import orthogonalize

pytestmark = pytest.mark.gpu

QUINTIC = (3.4445, -4.7750, 2.0315)


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


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [20, 33, 256, 300])
def test_updates_far_below_eps(dev, rows, dt):
    """|G| of 1e-8 .. 1e-30 with eps = 1e-7: X = G / (|G| + eps) is as small, and grows by a per step.
    The steps are all but linear there, so that a rounding of 2^-22 per step is passed on as it is: 2^-19 for the five."""
    make = torch.Generator().manual_seed(rows)
    base = torch.randn(rows, 320, generator=make)
    base /= base.norm()
    for size in (1e-8, 1e-12, 1e-13, 1e-14, 1e-15, 1e-20, 1e-30):
        g = (base * size).to(dt)
        for x in (g, g.t().contiguous()):
            want = iterate(x, [QUINTIC] * 5, 1e-7)
            got = orthogonalize(x.to(dev)).cpu().double()
            err = ((got - want).norm() / want.norm()).item()
            assert err <= 2.0**-19 + torch.finfo(dt).eps / 2, (size, tuple(x.shape), err)


def test_many_steps_from_far_below_eps_to_one(dev):
    """Forty steps take singular values from 1e-15 to 1: X is held at another scale in every step of the way up."""
    g = torch.randn(64, 200, generator=torch.Generator().manual_seed(4))
    g = g / g.norm() * 1e-22
    steps = [(3.0, -3.0, 1.0)] * 36 + [(1.875, -1.25, 0.375)] * 8
    got = orthogonalize(g.to(dev), coefficients=steps).cpu().double()
    u, _, v = torch.linalg.svd(g.double(), full_matrices=False)
    # the last steps converge to third order: what is left is their own roundings of X, A and B, 2^-22 each
    assert ((got - u @ v).norm() / 8.0).item() <= 2.0**-18


@pytest.mark.parametrize("steps", [[(1e-6, 0.0, 0.0), (1e6, 0.0, 0.0)], [(1e-10, 0.0, 0.0), (0.0, 1e30, 0.0)], [(1e-4, 0.0, 0.0), (0.0, 0.0, 1e20)],
                                   [(1e-9, 1e-9, 0.0), (1e9, -1e9, 1e9)]])
def test_steps_that_shrink_and_grow(dev, steps):
    """A step that makes all singular values small is known to do so: nothing is lost of the iterate.
    Roundings of 2^-22 of X, A and B, three products, slopes of five at most."""
    g = torch.randn(90, 140, generator=torch.Generator().manual_seed(5))
    want = iterate(g, steps, 0.0)
    got = orthogonalize(g.to(dev), coefficients=steps, eps=0.0).cpu().double()
    assert ((got - want).norm() / want.norm()).item() <= 9 * 5 * 2.0**-22


def test_one_call_with_tiny_usual_and_huge_updates(dev):
    base = [torch.randn(50 + 40 * i, 333, generator=torch.Generator().manual_seed(i)) for i in range(6)]
    mats = [b / b.norm() * s for b, s in zip(base, (1e-20, 1.0, 1e-9, 1e30, 0.0, 1e-13))]
    got = orthogonalize([m.to(dev) for m in mats])
    for m, o in zip(mats, got):
        want = iterate(m, [QUINTIC] * 5, 1e-7)
        assert (o.cpu().double() - want).norm() <= 1e-5 * want.norm()
        # alone it gets what it gets among others, but for the order of 32-bit sums
        assert ((orthogonalize(m.to(dev)) - o).double().norm() <= 1e-5 * o.double().norm()).item()
