# SPDX-License-Identifier: Apache-2.0
"""The orthogonalisation on the GPU against the iteration in 64 bits.

Tolerances, in the Frobenius norm relative to the result's: every product of one step is off by about
u = 2^-21 (two terms of fp16 carry 22 bits; sums in 32 bits) of its operands' norms, and what a step
leaves is amplified by at most a per following step where singular values are small.  Each step rounds X,
A and B (3 u), so that the error after n steps is at most 3 u (1 + a + ... + a^(n-1)) < 3 u a^n / (a - 1) times
the norm of X_k, |X_k|_2 <= 1.3 and |X_k|_F <= 1.3 sqrt(p): five steps of a = 3.4445 give 2^-21 * 3 * 485 * 1.4
= 1e-3 in the worst direction.  That bound needs all of the error to lie in directions whose singular values stay small;
relative to the whole norm the matrices below, none of whose singular values are that small, get a hundredth of it.
The result then rounds by half a step of its type (eps / 2 of each element, hence of the norm).
A last step in one fp16 term (bf16 results) adds 3 roundings of 2^-12 to X, A and B, each entering with a factor of
at most |a| + 3|b| + 5|c| < 28: below 3 * 28 * 2^-12 / sqrt(3) = 1.2e-2 at worst, and 3 * 2^-11 = 1.5e-3 as
independent errors of elements, which the test takes.
"""
import pytest
import torch

from fastsafetensors_amd import orthogonalize

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FIVE = [(3.4445, -4.7750, 2.0315)] * 5
POLAR = FIVE + [(1.875, -1.25, 0.375)] * 4
CORE = 1e-5          # the iteration itself (see above)
LAST_STEP = {"f32": 0.0, "f16": 0.0, "bf16": 1.5e-3}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def make(m, n, seed=0, scale=1e-3):
    g = torch.Generator().manual_seed(seed * 7919 + m * 131 + n)
    return torch.randn(m, n, generator=g) * scale


def iterate(g, coefficients=FIVE, eps=1e-7):
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + eps)
    for a, b, c in coefficients:
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
    return x.t() if flip else x


def check(got, g, dt, coefficients=FIVE, eps=1e-7, core=CORE, one_term=True):
    want = iterate(g, coefficients, eps)
    got = got.cpu().double()
    assert got.shape == want.shape and got.isfinite().all()
    tol = core + (LAST_STEP[dt] if one_term else 0.0) + torch.finfo(T[dt]).eps / 2
    err = ((got - want).norm() / want.norm().clamp_min(1e-30)).item()
    assert err <= tol, (tuple(g.shape), dt, err, tol)


SHAPES = [(1, 1), (1, 513), (700, 1), (2, 2), (5, 3), (31, 33), (64, 64), (65, 64), (77, 130), (128, 384), (129, 129), (260, 100), (300, 777)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_shapes_and_types(dev, dt):
    for i, (m, n) in enumerate(SHAPES):
        g = make(m, n, i).to(T[dt])
        got = orthogonalize(g.to(dev))
        assert got.dtype == g.dtype and got.is_contiguous()
        check(got, g, dt)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_slim_matrices(dev, dt):
    """Up to 32 rows or columns everything is done in 64 bits: what is left is the rounding of the result."""
    shapes = [(1, 1), (1, 2), (2, 1), (3, 255), (8, 256), (257, 9), (16, 16), (17, 4099), (5000, 31), (32, 32), (32, 70001), (100003, 2)]
    mats = [make(m, n, i).to(T[dt]) for i, (m, n) in enumerate(shapes)]
    for g, got in zip(mats, orthogonalize([g.to(dev) for g in mats], coefficients=POLAR)):
        want = iterate(g, POLAR)
        # half a step of the type of every element, and a 64-bit calculation's own 2^-40 or so of the largest
        assert ((got.cpu().double() - want).abs() <= want.abs() * (torch.finfo(T[dt]).eps / 2 * 1.001) + 2.0**-25 + want.abs().max() * 2.0**-40).all(), g.shape


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1024, 4096), (2048, 2048), (5000, 1100), (1500, 1500)])
def test_large_tiles(dev, dt, m, n):
    g = make(m, n).to(T[dt])
    check(orthogonalize(g.to(dev)), g, dt)


def test_one_step_matches_its_formula_closely(dev):
    """Every coefficient on its own: a X, A X and A^2 X."""
    for c in ((1.0, 0.0, 0.0), (0.0, 1.0, 0.0), (0.0, 0.0, 1.0), (-2.0, 0.5, 0.25)):
        for m, n in ((40, 40), (200, 333), (333, 200)):
            g = make(m, n)
            check(orthogonalize(g.to(dev), coefficients=[c]), g, "f32", [c], core=2e-6)


def test_the_result_is_orthogonal_with_enough_steps(dev):
    for m, n in ((96, 96), (100, 400), (400, 100)):
        g = torch.linalg.qr(make(max(m, n), min(m, n)))[0] @ torch.diag(torch.linspace(0.05, 1.0, min(m, n)))
        g = g if m > n else g.t()
        got = orthogonalize(g.to(dev), coefficients=POLAR).cpu().double()
        gram = got @ got.t() if m <= n else got.t() @ got
        # four steps of (15/8, -10/8, 3/8) take 1 + e to 1 + O(e^3): exact to the iteration's own error
        assert (gram - torch.eye(min(m, n))).abs().max() < 1e-4
        u, _, v = torch.linalg.svd(g.double(), full_matrices=False)
        assert (got - u @ v).abs().max() < 1e-4


def test_strong_directions_over_a_weak_floor(dev):
    """Spectra as momenta have them; here the core's error is amplified (ratio 1000: by a hundred)."""
    g = torch.Generator().manual_seed(3)
    u, v = torch.linalg.qr(torch.randn(256, 256, generator=g))[0], torch.linalg.qr(torch.randn(512, 256, generator=g))[0]
    s = torch.cat([torch.ones(8), torch.full((248,), 1e-3)])
    for dt in T:
        x = ((u * s) @ v.t()).to(T[dt])
        check(orthogonalize(x.to(dev)), x, dt, core=1e-4)


def test_scales_of_the_input(dev):
    """The norm is taken in 64 bits: squares of large or tiny elements do not leave the range."""
    for scale in (1e-30, 1e-20, 1.0, 1e20, 1e30):
        g = make(90, 120, scale=scale)
        check(orthogonalize(g.to(dev), eps=0.0), g, "f32", eps=0.0)
    g = make(64, 96)
    check(orthogonalize(g.to(dev), eps=0.5), g, "f32", eps=0.5, core=1e-4)  # eps of the norm's size: small singular values


def test_norms_that_32_bits_do_not_hold(dev):
    g = make(40, 90, 3, scale=1.0)
    for scale in (2.0**125, 2.0**-130):  # |G| is 2.5e39; and elements of a few denormal digits
        x = g * scale
        assert x.isfinite().all()
        check(orthogonalize(x.to(dev), eps=0.0), x, "f32", eps=0.0)


def test_zero_matrix_and_special_values(dev):
    assert (orthogonalize(torch.zeros(50, 70, device=dev)) == 0).all()
    for bad in (float("nan"), float("inf")):
        g = make(50, 70)
        g[3, 4] = bad
        clean = make(90, 30)
        got, other = orthogonalize([g.to(dev), clean.to(dev)])
        assert not got.isfinite().any() or got.isnan().any()
        check(other, clean, "f32")  # its neighbour in the call is untouched
    one = torch.zeros(200, 300)
    one[17, 23] = 5.0  # a single element: the largest entry an iterate can have
    got = orthogonalize(one.to(dev)).cpu()
    want = iterate(one)
    assert abs(got[17, 23].item() - want[17, 23].item()) < 1e-5 and got.count_nonzero() == 1


def test_batches_of_mixed_sizes_and_types(dev):
    mats = [make(1 + 37 * (i % 11), 1 + 53 * (i % 7), i).to(T[("f32", "f16", "bf16")[i % 3]]) for i in range(47)]
    mats[13], mats[29] = torch.zeros(0, 5), torch.zeros(8, 0, dtype=torch.bfloat16)
    got = orthogonalize([g.to(dev) for g in mats])
    for g, o in zip(mats, got):
        if g.numel():
            dt = next(k for k, t in T.items() if t == g.dtype)
            check(o, g, dt)
        else:
            assert o.shape == g.shape


def test_strides_pitch_and_in_place(dev):
    g = make(150, 90).to(torch.bfloat16)
    wide = torch.zeros(300, 400, dtype=torch.bfloat16, device=dev)
    wide[::2, 3:273:3] = g.to(dev)
    check(orthogonalize(wide[::2, 3:273:3]), g, "bf16")
    check(orthogonalize(g.t().contiguous().to(dev).t()), g, "bf16")
    check(orthogonalize(make(1, 90).to(torch.bfloat16).to(dev).expand(150, 90)), make(1, 90).to(torch.bfloat16).expand(150, 90), "bf16", core=1e-4)
    for at in range(4):  # rows of a wider tensor, at any element
        target = torch.full((150, 133), 3.0, dtype=torch.bfloat16, device=dev)
        out = target[:, at : at + 90]
        assert orthogonalize(g.to(dev), outs=out) is out
        check(out, g, "bf16")
        assert (target[:, :at] == 3).all() and (target[:, at + 90 :] == 3).all()
    flat = torch.empty(90, 150, dtype=torch.bfloat16, device=dev)
    orthogonalize([g.to(dev)], outs=[flat.t()])  # columns contiguous
    check(flat.t(), g, "bf16")
    x = g.to(dev)
    assert orthogonalize(x, outs=x) is x
    check(x, g, "bf16")


def slim_close(got, g, coefficients=FIVE):
    want = iterate(g, coefficients)  # 64 bits on both sides: half a step of the type, as in test_slim_matrices
    return ((got.cpu().double() - want).abs() <= want.abs() * (torch.finfo(g.dtype).eps / 2 * 1.001) + 2.0**-25 + want.abs().max() * 2.0**-40).all()


def test_more_slim_matrices_than_one_set_takes(dev):
    """Seventy of them between larger and empty ones: every second stored by columns, some pitched, all in place."""
    mats, kept = [], []
    for i in range(70):
        m, n, t = 1 + i * 5 % 32, 1 + i * 37 % 300, list(T)[i % 3]
        g = make(m, n, i).to(T[t]) if i % 4 < 2 else make(n, m, i).to(T[t])
        kept.append(g)
        held = torch.full((g.shape[0], g.shape[1] + i % 3), 7.0, dtype=g.dtype, device=dev)
        at = held[:, : g.shape[1]] if i % 2 else torch.empty(g.shape[::-1], dtype=g.dtype, device=dev).t()
        at.copy_(g)
        mats.append(at)
        if i % 20 == 0:
            mats += [torch.empty(0, 5, device=dev), make(100, 90, i).to(dev)]
            kept += [None, None]
    out = orthogonalize(mats, outs=mats)
    for at, g, o in zip(mats, kept, out):
        assert o is at and (g is None or slim_close(at, g)), at.shape
    held = torch.full((8, 40), 7.0, device=dev)
    orthogonalize([held[:, :33].copy_(make(8, 33))], outs=[held[:, :33]])
    assert (held[:, 33:] == 7.0).all()  # what lies between the rows stays


def test_special_values_in_slim_matrices(dev):
    g = make(12, 100, 5)
    assert torch.equal(orthogonalize(torch.zeros(12, 100, device=dev)).cpu(), torch.zeros(12, 100))
    assert orthogonalize(torch.zeros(12, 100, device=dev), eps=0.0).isnan().all()
    for bad in (float("inf"), float("nan")):
        b = g.clone()
        b[3, 77] = bad
        got = orthogonalize([b.to(dev), g.to(dev)])
        assert got[0].isnan().all() and slim_close(got[1], g)
    # squares of the largest floats do not overflow, nor do those of small ones vanish
    for scale in (2.0**124, 2.0**-100):
        got = orthogonalize((g * scale).to(dev), eps=0.0)
        assert ((got.cpu().double() - iterate(g, eps=0.0)).abs() <= 2.0**-24).all()


def test_slim_matrices_captured_and_replayed(dev):
    g = [make(32, 5000, 1).to(dev), make(900, 7, 2).to(dev)]
    out = [torch.empty_like(x) for x in g]
    orthogonalize(g, outs=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        orthogonalize(g, outs=out)
    for turn in range(3):
        for i, x in enumerate(g):
            x.copy_(make(*x.shape, 10 * turn + i))
        want = orthogonalize(g)
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want))


def test_column_blocks_of_one_tensor_in_place(dev):
    """The parts of a fused projection's update, each made orthogonal where it lies."""
    whole = make(96, 640, 41).to(dev)
    parts = whole.split([320, 192, 128], dim=1)
    want = orthogonalize([p.clone() for p in parts])
    got = orthogonalize(list(parts), outs=list(parts))
    for g, w, p in zip(got, want, whole.split([320, 192, 128], dim=1)):
        assert torch.equal(g, w) and torch.equal(p, w)


def test_the_result_does_not_depend_on_the_run_and_hardly_on_the_batch(dev):
    """Bit for bit the same from run to run; alone or among others the sums may be split differently, which
    is a difference in their 32-bit rounding only (and a step of the result's type where that decides)."""
    mats = [make(100 + 500 * i, 200, i).to(T[("f32", "bf16", "f16")[i % 3]]).to(dev) for i in range(7)]
    first = orthogonalize(mats)
    again = orthogonalize(mats)
    alone = [orthogonalize(g) for g in mats]
    for a, b, c in zip(first, again, alone):
        assert torch.equal(a, b)
        assert ((a.double() - c.double()).norm() / a.double().norm()).item() <= 1e-5 + torch.finfo(a.dtype).eps


def test_capture_and_replay(dev):
    mats = [torch.zeros(200, 300, device=dev), torch.zeros(130, 70, device=dev)]
    outs = [torch.empty_like(g) for g in mats]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        orthogonalize(mats, outs=outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        orthogonalize(mats, outs=outs)
    for turn in range(4):
        host = [make(*g.shape, seed=turn) for g in mats]
        for g, h in zip(mats, host):
            g.copy_(h.to(dev))
        graph.replay()
        torch.cuda.synchronize()
        eager = orthogonalize(mats)
        for o, e, h in zip(outs, eager, host):
            check(o, h, "f32")
            assert torch.equal(o, e)


def test_other_streams(dev):
    g = make(333, 444)
    x = g.to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = orthogonalize(x)
    here = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    check(got, g, "f32")
    assert torch.equal(got, here)


def test_refusals(dev):
    g = make(20, 30).to(dev)
    for error, match, args in ((TypeError, "update is", (g.double(),)), (ValueError, "two dimensions", (g[0],)),
                               (TypeError, "torch.Tensor", ([None],)), (RuntimeError, "requires a gradient", (g.clone().requires_grad_(),)),
                               (ValueError, "GPU memory", ([g, g.cpu()],))):
        with pytest.raises(error, match=match):
            orthogonalize(*args)
    with pytest.raises(ValueError, match="out is"):
        orthogonalize(g, outs=g.half())
    with pytest.raises(ValueError, match="overlap"):
        orthogonalize([g, g.clone()], outs=[torch.empty_like(g), g])
    with pytest.raises(ValueError, match="overlap"):
        out = torch.empty_like(g)
        orthogonalize([g, g.clone()], outs=[out, out])
    with pytest.raises(ValueError, match="rows or contiguous columns"):
        orthogonalize(g, outs=torch.empty(40, 60, device=dev)[::2, ::2])
    with torch.no_grad():
        orthogonalize(g.clone().requires_grad_())
