# SPDX-License-Identifier: Apache-2.0
"""The orthogonalisation of updates whose weight sits in a few rows, elements or directions.

Nothing averages a rounding that meets one strong element, so these show what flat spectra hide.

Tolerances, Frobenius norm relative to the 64-bit result's.  Iterates held as two fp16 terms round by 2^-22 of
a value at most, products leave out 2^-22, fp32 rounds by 2^-24, sums are the same 32 bits: the iteration may
be off by four times what the plain 32-bit form is off by.  That form can be lucky where only a few
numbers are not zero; one number alone is perturbed, per step, by a rounding of X, A and B and by what three
products leave out, with factors of |b| + 2 |c| = 9 at most for A, 7 for B: about 5 * 2^-22 as independent
errors, and behind five steps, whose slopes at 0.7 .. 1.2 are 1.6 or so, three times that: 2^-18 is allowed at least.
Rounding the result to its type then costs what it costs the 64-bit result, plus the distance between the
two before rounding (the distance to the nearest representable value changes by at most that)."""
import pytest
import torch

from fastsafetensors_amd import orthogonalize

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FIVE = [(3.4445, -4.7750, 2.0315)] * 5
POLAR = FIVE + [(1.875, -1.25, 0.375)] * 4


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def make(kind, m, n, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + m * 131 + n)
    x = torch.randn(m, n, generator=g)
    if kind == "flat":
        return x * 1e-3
    if kind == "one row":
        out = torch.zeros(m, n)
        out[m // 3] = x[0]
        return out
    if kind == "strong row":
        x *= 0.01
        x[m // 3] *= 100
        return x
    if kind == "strong row and column":
        x *= 0.01
        x[m // 3] *= 100
        x[:, n // 5] *= 100
        return x
    if kind == "hot rows":
        x[:: m // 8] *= 1000
        return x
    if kind == "one element":
        out = torch.zeros(m, n)
        out[m // 3, n // 5] = 0.37
        return out
    if kind == "diagonal":
        out = torch.zeros(m, n)
        out.diagonal().copy_(torch.where(torch.arange(min(m, n)) < 8, 1.0, 1e-3))
        return out
    left, right = torch.randn(m, 8, generator=g), torch.randn(8, n, generator=g)
    if kind == "rank 8":
        return left @ right
    assert kind == "spiked"
    return left @ right / (m * n) ** 0.5 + 1e-3 * x / (m**0.5 + n**0.5)


def iterate(x, coefficients, eps=1e-7):
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    x = x / (x.square().sum().sqrt() + eps)
    for a, b, c in coefficients:
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if flip else x


def check(dev, g, coefficients, what, at_least=2.0**-18):
    g = g.to(dev)
    want = iterate(g.double(), coefficients)
    size = want.norm()
    core = max(4 * ((iterate(g.float(), coefficients).double() - want).norm() / size).item(), at_least)
    tol = core if g.dtype == torch.float32 else 2 * core + ((want.to(g.dtype).double() - want).norm() / size).item()
    got = orthogonalize(g, coefficients=coefficients).double()
    err = ((got - want).norm() / size).item()
    print(f"{what}: {err:.3g}, allowed {tol:.3g}", flush=True)
    assert err <= tol, (what, err, tol)


KINDS = ["flat", "one row", "strong row", "strong row and column", "hot rows", "one element", "diagonal", "rank 8", "spiked"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt,m,n", [("f32", 2560, 2560), ("f32", 2500, 2600), ("f16", 768, 768), ("f16", 600, 900), ("f16", 900, 600),
                                    ("bf16", 768, 768), ("bf16", 1100, 2000)])
def test_spectra(dev, kind, dt, m, n):
    check(dev, make(kind, m, n).to(T[dt]), FIVE, (kind, dt, m, n))


@pytest.mark.parametrize("kind", ["one row", "strong row", "rank 8"])
@pytest.mark.parametrize("dt,m,n", [("f32", 2560, 2560), ("bf16", 768, 768)])
def test_spectra_with_the_steps_that_end_at_one(dev, kind, dt, m, n):
    check(dev, make(kind, m, n).to(T[dt]), POLAR, (kind, dt, m, n))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_a_step_whose_product_is_the_whole_result(dev, dt):
    """a = 0: X' = A X is 1 / p of X's size.  Elements are held to 2^-24 of the iterates' typical element at the start,
    when |X|_F = 1: 2^-24 / |X'|_F of the result, which the second step (a = 1.5) passes on."""
    g = make("flat", 600, 600).to(T[dt])
    shrunk = iterate(g.double(), [(0.0, 1.0, 0.0)]).norm().item()
    check(dev, g, [(0.0, 1.0, 0.0), (1.5, -0.5, 0.0)], dt, at_least=2.0**-24 / shrunk)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_results_below_512_rows_are_off_by_their_rounding(dev, dt):
    for kind in ("flat", "strong row", "rank 8"):
        check(dev, make(kind, 300, 444).to(T[dt]), FIVE, (kind, dt))
