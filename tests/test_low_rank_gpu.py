# SPDX-License-Identifier: Apache-2.0
"""The low-rank merge on the GPU against the formula in 64 bits.

Tolerance of one element, from the arithmetic: the sum of r products (times the products of the split)
is accumulated in fp32, each addition off by at most one unit in the last place (2^-23) of a
partial sum that is at most S = |s| sum |u d|; splitting fp32 factors leaves out less than 2^-16 S with two bf16
terms (three parts of 2^-18) and 2^-24 S with three; adding the weight rounds once more (2^-24); and the
result is off by half a step of its type (finfo.eps / 2 of its magnitude, or half the smallest subnormal).
"""
import pytest
import torch

from fastsafetensors_amd import LowRankUpdate, merge_low_rank

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
HALF_SUBNORMAL = {"f32": 2.0**-150, "f16": 2.0**-25, "bf16": 2.0**-134, "e4m3": 2.0**-10}
ONE_TERM = {("bf16", "bf16"), ("f16", "f16")}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def make(m, n, r, wt, ut, dt, seed=0):
    g = torch.Generator().manual_seed(seed * 1000003 + m * 1009 + n * 31 + r)
    w = torch.randn(m, n, generator=g) * (30.0 if wt == "e4m3" else 0.05)
    u, d = torch.randn(m, r, generator=g) * 0.3, torch.randn(r, n, generator=g) * 0.3
    return w.to(T[wt]), u.to(T[ut]), d.to(T[dt])


def check(got, w, u, d, s, wt, ut, dt, ws=None):
    """``got`` (on the GPU) against w + s u d of the host tensors, in 64 bits (there, too)."""
    w64, u64, d64 = (t.to(got.device).double() for t in (w, u, d))
    ws = None if ws is None else ws.to(got.device)
    held = torch.ones((), device=got.device) if ws is None else ws.double().reshape(-1, 1) if ws.numel() > 1 else ws.double().reshape(())
    want = w64 + s * (u64 @ d64) / held
    bound = abs(s) * (u64.abs() @ d64.abs()) / held
    r = u.shape[1]
    products = 1 if (ut, dt) in ONE_TERM else 6 if wt == "f32" else 3
    split = 0.0 if (ut, dt) in ONE_TERM else 2.0**-24 if wt == "f32" else 2.0**-16
    slack = bound * ((r * products + 4) * 2.0**-23 + split) + (want.abs() + w64.abs()) * 2.0**-23
    if wt == "e4m3":
        want = want.clamp(-448.0, 448.0)
    tol = (want.abs() + slack) * (torch.finfo(T[wt]).eps / 2) + HALF_SUBNORMAL[wt] + slack
    got = got.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), (got - want)[bad][:4], tol[bad][:4])


SHAPES = [(1, 1), (1, 4095), (511, 1), (3, 5), (64, 64), (65, 63), (128, 192), (129, 1025), (200, 767), (1000, 72)]


@pytest.mark.parametrize("wt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("ut,dt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "bf16")])
def test_shapes_types_and_ranks(dev, wt, ut, dt):
    for k, (m, n) in enumerate(SHAPES):
        for r in ((1, 5, 32) if k % 2 else (8, 33, 64)):
            w, u, d = make(m, n, r, wt, ut, dt)
            ws = None
            if wt == "e4m3":
                ws = torch.tensor(0.37) if k % 3 else torch.rand(m) + 0.5
            s = (1.0, -0.75, 2.0)[k % 3]
            g = LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), s, None if ws is None else ws.to(dev))
            (got,) = merge_low_rank([g])
            assert got is g.weight
            check(got, w, u, d, s, wt, ut, dt, ws)


@pytest.mark.parametrize("wt", ["f32", "bf16", "e4m3"])
def test_large_ranks_and_many_tiles(dev, wt):
    for m, n, r in ((1024, 1536, 256), (300, 333, 1000), (2500, 4096, 16)):
        w, u, d = make(m, n, r, wt, "bf16", "bf16")
        ws = torch.tensor(2.5) if wt == "e4m3" else None
        (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 0.5, None if ws is None else ws.to(dev))])
        check(got, w, u, d, 0.5, wt, "bf16", "bf16", ws)


@pytest.mark.parametrize("ut,dt", [("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("wt", ["f32", "f16", "bf16", "e4m3"])
def test_ranks_that_go_through_shared_operands(dev, wt, ut, dt):
    """Ranks from the first that the walking kernel leaves to another on, with edges on both sides."""
    for m, n, r in ((1, 300, 97), (129, 1, 160), (130, 517, 161), (257, 255, 449), (300, 333, 1000)):
        w, u, d = make(m, n, r, wt, ut, dt)
        ws = torch.rand(m) + 0.5 if wt == "e4m3" else None
        (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 0.5, None if ws is None else ws.to(dev))])
        check(got, w, u, d, 0.5, wt, ut, dt, ws)


@pytest.mark.parametrize("r", [5, 33])
@pytest.mark.parametrize("wt", ["f32", "f16", "bf16", "e4m3"])
def test_long_walks_with_edges(dev, wt, r):
    """More tiles than the one-launch kernel takes: walks of several tiles, the last panel and the last tile of each cut off."""
    n = {"f32": 2047, "f16": 4095, "bf16": 4095, "e4m3": 8189}[wt]
    w, u, d = make(5003, n, r, wt, "bf16", "bf16")
    ws = torch.rand(5003) + 0.5 if wt == "e4m3" else None
    (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 0.5, None if ws is None else ws.to(dev))])
    check(got, w, u, d, 0.5, wt, "bf16", "bf16", ws)
    w, u, d = make(5056, n + 64 - n % 64, r, wt, "bf16", "bf16")  # ... and whole lines throughout
    (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 0.5, None if ws is None else torch.ones(1, device=dev))])
    check(got, w, u, d, 0.5, wt, "bf16", "bf16", None if ws is None else torch.ones(1))


@pytest.mark.parametrize("wt", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("r", [7, 40, 200])
def test_pitched_and_misaligned_weights_leave_their_surroundings_alone(dev, wt, r):
    """A column block of a wider tensor at every element offset of a 16-byte vector, in place and out of place."""
    m, n, size = 70, 131, T[wt].itemsize
    w, u, d = make(m, n, r, wt, "bf16", "bf16")
    ws = torch.tensor(1.25) if wt == "e4m3" else None
    wsd = None if ws is None else ws.to(dev)
    for at in range(0, 16 // size, 1 if size > 1 else 5):
        whole = torch.full((m, n + 37), 7.0).to(T[wt]).to(dev)
        before = whole.view(torch.uint8).clone()
        block = whole[:, at : at + n]
        block.copy_(w.to(dev))
        target = torch.full((m, n + 21), 3.0).to(T[wt]).to(dev)
        out = target[:, 2 : 2 + n]
        merge_low_rank([LowRankUpdate(block, u.to(dev), d.to(dev), 1.5, wsd, out)])
        check(out, w, u, d, 1.5, wt, "bf16", "bf16", ws)
        assert torch.equal(block.cpu().view(torch.uint8), w.view(torch.uint8))  # the source is as it was
        assert (target[:, :2].float() == 3).all() and (target[:, 2 + n :].float() == 3).all()
        merge_low_rank([LowRankUpdate(block, u.to(dev), d.to(dev), 1.5, wsd)])
        check(block, w, u, d, 1.5, wt, "bf16", "bf16", ws)
        after = whole.view(torch.uint8).clone()
        after[:, at * size : (at + n) * size] = before[:, at * size : (at + n) * size]
        assert torch.equal(after, before)


def test_strided_and_broadcast_factors_and_weights_stored_by_columns(dev):
    m, n, r = 150, 90, 12
    w, u, d = make(m, n, r, "bf16", "f32", "f32")
    wide_u, wide_d = torch.zeros(m, 3 * r), torch.zeros(2 * r, n)
    wide_u[:, ::3], wide_d[1::2] = u, d
    for up in (u.to(dev), u.t().contiguous().to(dev).t(), wide_u.to(dev)[:, ::3]):
        for down in (d.to(dev), d.t().contiguous().to(dev).t(), wide_d.to(dev)[1::2]):
            (got,) = merge_low_rank([LowRankUpdate(w.to(dev), up, down, 0.5)])
            check(got, w, u, d, 0.5, "bf16", "f32", "f32")
    col = w.t().contiguous().to(dev).t()  # columns contiguous
    (got,) = merge_low_rank([LowRankUpdate(col, u.to(dev), d.to(dev), 0.5)])
    assert got is col and col.stride() == (1, m)
    check(col, w, u, d, 0.5, "bf16", "f32", "f32")
    one = u[:, :1].to(dev).expand(m, r)  # stride 0
    (got,) = merge_low_rank([LowRankUpdate(w.to(dev), one, d.to(dev), 0.5)])
    check(got, w, u[:, :1].expand(m, r), d, 0.5, "bf16", "f32", "f32")


def test_many_weights_of_all_kinds_in_one_call(dev):
    """More jobs than one launch holds, every kernel variant, empty ones in between."""
    updates, want = [], []
    for i in range(90):
        wt = ("f32", "f16", "bf16", "e4m3")[i % 4]
        ut, dt = (("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"))[i % 3]
        m, n, r = (0 if i % 17 == 5 else 1 + 7 * i), (0 if i % 19 == 7 else 300 - 3 * i), (0 if i % 23 == 9 else i % 40)
        w, u, d = make(m, n, r, wt, ut, dt, seed=i)
        ws = torch.tensor(0.8) if wt == "e4m3" else None
        updates.append(LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 0.25, None if ws is None else ws.to(dev)))
        want.append((w, u, d, 0.25, wt, ut, dt, ws))
    got = merge_low_rank(updates)
    for t, args in zip(got, want):
        check(t, *args)


def test_rank_zero_and_scale_zero_keep_every_weight(dev):
    for wt in T:
        w, u, d = make(65, 70, 0, wt, "bf16", "bf16")
        out = torch.zeros(65, 70).to(T[wt]).to(dev)
        ws = torch.tensor(0.3, device=dev) if wt == "e4m3" else None
        merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 3.0, ws, out)])
        assert torch.equal(out.cpu().view(torch.uint8), w.view(torch.uint8)), wt
        w, u, d = make(65, 70, 9, wt, "bf16", "bf16")
        x = w.to(dev)
        merge_low_rank([LowRankUpdate(x, u.to(dev), d.to(dev), 0.0, ws)])
        assert torch.equal(x.cpu().float(), w.float()), wt


def test_special_values(dev):
    inf, nan = float("inf"), float("nan")
    for wt in ("f32", "f16", "bf16"):
        w, u, d = make(80, 80, 4, wt, "f32", "f32")
        w[3, 5], w[4, 6], w[5, 7] = inf, -inf, nan
        (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 1.0)])
        got = got.cpu()
        assert got[3, 5] == inf and got[4, 6] == -inf and got[5, 7].isnan()
        assert got.isfinite().sum() == 80 * 80 - 3
        # a factor that is not finite spoils its row, and nothing else
        w, u, d = make(80, 80, 4, wt, "f32", "f32")
        u[11, 2] = nan
        (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 1.0)])
        got = got.cpu()
        assert got[11].isnan().all() and got.isfinite().sum() == 79 * 80
        # fp32 factors beyond bf16's largest value are split without overflow (the smaller factor's second
        # term is below the normal range and may be lost: 2^-9 of it)
        big = torch.full((8, 1), 3.4e38)
        tiny = torch.full((1, 8), 2e-38)
        (got,) = merge_low_rank([LowRankUpdate(torch.zeros(8, 8, dtype=T[wt], device=dev), big.to(dev), tiny.to(dev), 1.0)])
        assert torch.allclose(got.cpu().float(), torch.full((8, 8), 6.8), rtol=2**-7, atol=0)


def test_fp8_saturates_and_keeps_nan(dev):
    w = torch.tensor([[448.0, -448.0, 96.0, 0.0]]).to(torch.float8_e4m3fn)
    w.view(torch.uint8)[0, 3] = 0x7F
    u, d = torch.full((1, 1), 1.0), torch.tensor([[1000.0, -1000.0, 5.0, 1.0]])
    (got,) = merge_low_rank([LowRankUpdate(w.to(dev), u.to(dev), d.to(dev), 1.0, torch.ones(1, device=dev))])
    got = got.cpu().float()
    assert got[0, :3].tolist() == [448.0, -448.0, 104.0]  # 101 lies between 96 and 104
    assert got[0, 3].isnan()


def test_streams_and_other_current_stream(dev):
    w, u, d = make(700, 900, 16, "bf16", "bf16", "bf16")
    x, ud, dd = w.to(dev), u.to(dev), d.to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            out = torch.empty_like(x)
            merge_low_rank([LowRankUpdate(x, ud, dd, 0.5, out=out)])
    torch.cuda.current_stream().wait_stream(side)
    check(out, w, u, d, 0.5, "bf16", "bf16", "bf16")


def test_capture_and_replay(dev):
    """Two graphs over the same weights, replayed in turn with eager work between."""
    w, u, d = make(300, 500, 20, "bf16", "f32", "f32")
    x, ud, dd = w.to(dev), u.to(dev), d.to(dev)
    outs = [torch.empty_like(x), torch.empty_like(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        merge_low_rank([LowRankUpdate(x, ud, dd, 0.5, out=outs[0])])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s, out in zip((0.5, -1.0), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            merge_low_rank([LowRankUpdate(x, ud, dd, s, out=out)])
        graphs.append(graph)
    for turn in range(4):
        g = torch.Generator().manual_seed(turn)
        u = torch.randn(u.shape, generator=g) * 0.2
        ud.copy_(u.to(dev))
        for graph, out, s in zip(graphs, outs, (0.5, -1.0)):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            check(out, w, u, d, s, "bf16", "f32", "f32")
            (eager,) = merge_low_rank([LowRankUpdate(x, ud, dd, s, out=torch.empty_like(x))])
            assert torch.equal(eager, out)


def test_refusals(dev):
    w, u, d = (t.to(dev) for t in make(20, 30, 4, "bf16", "bf16", "bf16"))

    def refused(error, match, *args, **kw):
        before = w.clone()
        with pytest.raises(error, match=match):
            merge_low_rank([LowRankUpdate(*args, **kw)])
        assert torch.equal(w, before)

    refused(TypeError, "weight is", w.double(), u, d)
    refused(TypeError, "up is", w, u.double(), d)
    refused(TypeError, "down is", w, u, d.to(torch.float8_e4m3fn))
    refused(ValueError, "two dimensions", w[0], u, d)
    refused(ValueError, "shapes do not match", w, u[:, :3], d)
    refused(ValueError, "shapes do not match", w, u, d[:, :3])
    refused(ValueError, "out is", w, u, d, out=w.float())
    refused(ValueError, "weight_scale goes with", w, u, d, weight_scale=torch.ones(1, device=dev))
    refused(ValueError, "needs its weight_scale", w.to(torch.float8_e4m3fn), u, d)
    refused(TypeError, "not fp32", w.to(torch.float8_e4m3fn), u, d, weight_scale=torch.ones(1, device=dev, dtype=torch.bfloat16))
    refused(ValueError, "neither one value", w.to(torch.float8_e4m3fn), u, d, weight_scale=torch.ones(3, device=dev))
    refused(ValueError, "GPU memory", w, u.cpu(), d)
    refused(ValueError, "contiguous rows", torch.zeros(40, 60, device=dev, dtype=torch.bfloat16)[::2, ::2], u, d)
    refused(ValueError, "overlap", torch.zeros(1, 30, device=dev, dtype=torch.bfloat16).expand(20, 30), u, d)
    refused(RuntimeError, "requires a gradient", w, u.clone().requires_grad_(), d)
    with pytest.raises(ValueError, match="overlap"):
        merge_low_rank([LowRankUpdate(w, u, d), LowRankUpdate(w, u, d)])
    for scale in (float("inf"), float("nan"), 1e39):
        refused(ValueError, "finite", w, u, d, scale=scale)
        refused(ValueError, "finite", w, u, d, scale=scale, out=torch.empty_like(w))
    leaf = u.clone().requires_grad_()
    with torch.no_grad():
        merge_low_rank([LowRankUpdate(w, leaf, d)])


def test_a_merge_in_place_is_seen_by_autograd(dev):
    """A weight that a recorded product still needs must not change unnoticed."""
    w, u, d = (t.to(dev) for t in make(20, 30, 4, "f32", "f32", "f32"))
    x = torch.randn(5, 20, device=dev, requires_grad=True)
    y = (x @ w).sum()
    merge_low_rank([LowRankUpdate(w, u, d)])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_from_plain_c():
    """A C99 program with no Python, torch or C++ in it merges and orthogonalises and checks the results on the host."""
    import os
    import subprocess

    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cabi_update", "cabi_update.bin")
    if not os.path.exists(exe):
        pytest.skip("tests/cabi_update/cabi_update.bin is not built (run __graft_entry__.build())")
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "cabi_update: ok" in run.stdout, run.stdout + run.stderr
