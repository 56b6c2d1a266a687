# SPDX-License-Identifier: Apache-2.0
"""Adapter files and fine-tuned checkpoints merged into a loaded one, from disk to the shards a rank takes."""
import pytest
import torch

from fastsafetensors_amd import SafeTensorsFileLoader, SingleGroup, StubProcessGroup, DType
from fastsafetensors_amd import checkpoints as ck
from fastsafetensors_amd.checkpoints import TensorSpec, write_checkpoint

pytestmark = pytest.mark.gpu

PREFIX = "base_model.model."


def write(path, specs, seed):
    kept = {}

    def keep(spec, chunk):
        kept.setdefault(spec.name, []).append(chunk.clone())

    write_checkpoint(str(path), specs, seed, on_chunk=keep, pad_rem=2)
    return {k: torch.cat(v) if v[0].dim() else v[0] for k, v in kept.items()}


def pair(module, out_features, in_features, r, dtype, infix=""):
    return [TensorSpec(f"{PREFIX}{module}.lora_A{infix}.weight", dtype, (r, in_features)),
            TensorSpec(f"{PREFIX}{module}.lora_B{infix}.weight", dtype, (out_features, r))]


def load(path, pg=None, **kw):
    pg = pg or SingleGroup()
    loader = SafeTensorsFileLoader(pg, "cuda:0", max_threads=4, disable_cache=kw.pop("disable_cache", True))
    loader.add_filenames({pg.rank(): [str(path)]})
    return loader, loader.copy_files_to_device(**kw)


def merged64(w, a, b, s, held=1.0):
    return (w.double() * held + s * (b.double() @ a.double())) / held


def close(got, want, dtype, w, a, b, s):
    """Half a step of the type on top of what the sum in 32 bits is off by: each of its r (times three, where
    fp32 factors are split into two terms) additions rounds a partial sum of at most S = |s| sum |b||a| by
    2^-23 at most, the split leaves out less than 2^-16 S (16-bit weights; fp16 and bf16 factors are not
    split), and adding the weight rounds by 2^-24 of the result and of the weight it cancels with."""
    S = abs(s) * (b.double().abs() @ a.double().abs())
    S = S if S.shape == w.shape else S.t()
    split = a.dtype == torch.float32
    slack = S * ((a.shape[0] * (3 if split else 1) + 4) * 2.0**-23 + (2.0**-16 if split else 0.0)) + (want.abs() + w.double().abs()) * 2.0**-23
    return (got.cpu().double() - want).abs() - slack <= (want.abs() + slack) * (torch.finfo(dtype).eps / 2)


def test_a_layer_is_merged_in_place_and_then_cut_for_a_rank(tmp_path):
    base = ck.llama_layer_specs(0, 256, 64, 688, DType.BF16)
    modules = {"model.layers.0.self_attn.q_proj": (256, 256), "model.layers.0.self_attn.k_proj": (64, 256),
               "model.layers.0.mlp.down_proj": (256, 688)}
    specs = [s for m, (o, i) in modules.items() for s in pair(m, o, i, 8, DType.F32, ".default")]
    w = write(tmp_path / "base.safetensors", base, 1)
    ab = write(tmp_path / "adapter.safetensors", specs, 2)
    l0, bufs = load(tmp_path / "base.safetensors", StubProcessGroup(1, 2), disable_cache=False)
    l1, adapter = load(tmp_path / "adapter.safetensors")
    q = "model.layers.0.self_attn.q_proj.weight"
    old = bufs.get_sharded(q, 0).clone()  # kept by the loader: disable_cache=False
    names = bufs.merge_adapter(adapter, alpha=400.0, scale=None)
    assert sorted(names) == sorted(f"{m}.weight" for m in modules)
    for m in modules:
        a, b = ab[f"{PREFIX}{m}.lora_A.default.weight"], ab[f"{PREFIX}{m}.lora_B.default.weight"]
        want = merged64(w[f"{m}.weight"], a, b, 50.0)
        dim = 1 if "down" in m else 0
        half = want.shape[dim] // 2
        got = torch.zeros_like(w[f"{m}.weight"])
        got.narrow(dim, half, half).copy_(bufs.get_sharded(f"{m}.weight", dim))
        assert close(got, want, torch.bfloat16, w[f"{m}.weight"], a, b, 50.0).narrow(dim, half, half).all(), m
    assert not torch.equal(bufs.get_sharded(q, 0), old)
    for name in w:  # everything else is as the file has it
        if name not in names:
            assert torch.equal(bufs.get_sharded(name, -1).cpu(), w[name]), name
    for x in (bufs, adapter, l0, l1):
        x.close()


def test_fan_in_fan_out_and_downcast_on_load(tmp_path):
    base = ck.gpt2_specs(1, 96, 100, 32, DType.F32)
    spec = TensorSpec("h.0.attn.c_attn.weight", DType.F32, (96, 288))
    assert any(s.name == spec.name and tuple(s.shape) == spec.shape for s in base)
    w = write(tmp_path / "base.safetensors", base, 3)
    ab = write(tmp_path / "adapter.safetensors", pair("h.0.attn.c_attn", 288, 96, 4, DType.F16), 4)
    a, b = (ab[f"{PREFIX}h.0.attn.c_attn.lora_{k}.weight"] for k in "AB")
    for dtype, t in ((DType.AUTO, torch.float32), (DType.BF16, torch.bfloat16)):
        l0, bufs = load(tmp_path / "base.safetensors", dtype=dtype)
        l1, adapter = load(tmp_path / "adapter.safetensors")
        view = bufs.get_tensor(spec.name)
        assert bufs.merge_adapter(adapter, scale=3.0, fan_in_fan_out=True) == [spec.name]
        start = w[spec.name].to(t)
        want = start.double() + 3.0 * (b.double() @ a.double()).t()
        assert view.dtype == t and close(view, want, t, start, a, b, 3.0).all()  # the view shows the merged weight
        assert bufs.merge_adapter(adapter, scale=-3.0, fan_in_fan_out=True) == [spec.name]
        assert (view.cpu() - start).abs().max() <= 2 * torch.finfo(t).eps * want.abs().max()  # two roundings
        for x in (bufs, adapter, l0, l1):
            x.close()


def test_fp8_weights_keep_their_scale(tmp_path):
    base = ck.llama_layer_specs(0, 128, 32, 272, DType.BF16, fp8=True)
    m = "model.layers.0.mlp.gate_proj"
    w = write(tmp_path / "base.safetensors", base, 5)
    ab = write(tmp_path / "adapter.safetensors", pair(m, 272, 128, 16, DType.BF16), 6)
    l0, bufs = load(tmp_path / "base.safetensors")
    l1, adapter = load(tmp_path / "adapter.safetensors")
    assert bufs.merge_adapter(adapter, alpha=32.0) == [f"{m}.weight"]
    held = w[f"{m}.weight_scale"].double()
    want = merged64(w[f"{m}.weight"], ab[f"{PREFIX}{m}.lora_A.weight"], ab[f"{PREFIX}{m}.lora_B.weight"], 2.0, held)
    got = bufs.get_tensor(f"{m}.weight")
    assert got.dtype == torch.float8_e4m3fn
    # half a step of e4m3 (2^-4, 2^-10 below its normal range) and a little for the fp32 sum
    assert ((got.cpu().double() - want).abs() <= want.abs() * (2.0**-4 + 2.0**-18) + 2.0**-10).all()
    assert torch.equal(bufs.get_tensor(f"{m}.weight_scale").cpu(), w[f"{m}.weight_scale"])
    for x in (bufs, adapter, l0, l1):
        x.close()


def test_adapters_that_do_not_fit_change_nothing(tmp_path):
    base = [TensorSpec("a.weight", DType.BF16, (64, 32)), TensorSpec("b.weight", DType.BF16, (64, 32))]
    w = write(tmp_path / "base.safetensors", base, 7)
    good = pair("a", 64, 32, 4, DType.BF16)
    cases = {
        "not a lora_A": good + [TensorSpec(f"{PREFIX}a.lora_magnitude_vector", DType.BF16, (64,))],
        "only one of": good + pair("b", 64, 32, 4, DType.BF16)[:1],
        "was not found": good + pair("c", 64, 32, 4, DType.BF16),
        "do not match": good + pair("b", 64, 31, 4, DType.BF16),
        "more than one": good + pair("a", 64, 32, 4, DType.BF16, ".other"),
        "two dimensions": good + [TensorSpec(f"{PREFIX}b.lora_A.weight", DType.BF16, (4,)), TensorSpec(f"{PREFIX}b.lora_B.weight", DType.BF16, (64, 4))],
    }
    l0, bufs = load(tmp_path / "base.safetensors")
    for i, (match, specs) in enumerate(cases.items()):
        write(tmp_path / f"{i}.safetensors", specs, 8)
        l1, adapter = load(tmp_path / f"{i}.safetensors")
        with pytest.raises(ValueError, match=match):
            bufs.merge_adapter(adapter, scale=1.0)
        for bad in (dict(), dict(scale=1.0, alpha=2.0)):
            with pytest.raises(ValueError, match="either alpha or scale"):
                bufs.merge_adapter(adapter, **bad)
        adapter.close()
        l1.close()
    for name in w:
        assert torch.equal(bufs.get_tensor(name).cpu(), w[name])
    bufs.close()
    l0.close()


def polar(d):
    u, s, v = torch.linalg.svd(d, full_matrices=False)
    return u @ v, s.mean()


def test_fine_tuned_checkpoints_are_merged_with_orthogonalised_updates(tmp_path):
    shapes = {"model.a.weight": (96, 64), "model.b.weight": (64, 160), "model.norm.weight": (64,), "model.embed.weight": (50, 64)}
    specs = [TensorSpec(n, DType.F32, s) for n, s in shapes.items()]
    base = write(tmp_path / "base.safetensors", specs + [TensorSpec("other.weight", DType.F32, (7, 7))], 10)
    tuned = [write(tmp_path / f"t{i}.safetensors", specs, 20 + i) for i in range(3)]  # as far from the base as from each other
    l0, bufs = load(tmp_path / "base.safetensors")
    loaded = [load(tmp_path / f"t{i}.safetensors") for i in range(3)]
    names = bufs.merge_checkpoints([b for _, b in loaded], scale=0.5, orthogonal=["model.a.weight", "model.b.weight"])
    assert sorted(names) == sorted(shapes)
    for n in shapes:
        d = sum(t[n].double() - base[n].double() for t in tuned)
        got = bufs.get_tensor(n).cpu().double()
        if n in ("model.a.weight", "model.b.weight"):
            o, s = polar(d)
            # The update's singular values lie within a factor of a few hundred, which the nine steps take to 1 within
            # 1e-3 at the lower end and 1e-5 elsewhere; entries of o are about 0.1, s about 0.5.
            assert (got - (base[n].double() + 0.5 * s * o)).abs().max() < 1e-3 * s, n
        else:
            assert (got - (base[n].double() + 0.5 * d / 3)).abs().max() < 4 * 2.0**-24 * 0.5, n  # a few roundings of values below 0.5
    assert torch.equal(bufs.get_tensor("other.weight").cpu(), base["other.weight"])
    for x in (bufs, l0, *(y for pair_ in loaded for y in pair_)):
        x.close()


def test_checkpoints_that_do_not_fit_change_nothing(tmp_path):
    base = write(tmp_path / "base.safetensors", [TensorSpec("a", DType.BF16, (8, 8)), TensorSpec("b", DType.BF16, (8,))], 1)
    bad = {"x": ("was not found", [TensorSpec("c", DType.BF16, (8, 8))]), "y": ("shapes do not match", [TensorSpec("a", DType.BF16, (8, 9))]),
           "z": ("of one type", [TensorSpec("b", DType.BF16, (8,)), TensorSpec("a", DType.F16, (8, 8))])}
    l0, bufs = load(tmp_path / "base.safetensors")
    for key, (match, specs) in bad.items():
        write(tmp_path / f"{key}.safetensors", specs, 2)
        l1, other = load(tmp_path / f"{key}.safetensors")
        with pytest.raises((ValueError, TypeError), match=match):
            bufs.merge_checkpoints([other])
        other.close()
        l1.close()
    write(tmp_path / "good.safetensors", [TensorSpec("a", DType.BF16, (8, 8))], 3)
    l1, good = load(tmp_path / "good.safetensors")
    for args in (([],), ([good], 1.0, ["nowhere"])):
        with pytest.raises(ValueError):
            bufs.merge_checkpoints(*args)
    for n in base:
        assert torch.equal(bufs.get_tensor(n).cpu(), base[n])
    assert bufs.merge_checkpoints([good], scale=0.0) == ["a"]
    assert torch.equal(bufs.get_tensor("a").cpu(), base["a"])
    for x in (bufs, good, l0, l1):
        x.close()


def test_checkpoints_then_an_adapter_then_a_rank_s_shards(tmp_path):
    """Both operators on one loaded file, as a server that specialises a base checkpoint uses them: fine-tuned checkpoints merged in,
    an adapter merged on top, the adapter taken out again, a rank's block cut -- on a stream of its own, without a synchronisation."""
    shapes = {"q.weight": (192, 128), "down.weight": (96, 320)}
    specs = [TensorSpec(n, DType.F32, s) for n, s in shapes.items()]
    base = write(tmp_path / "base.safetensors", specs, 30)
    tuned = write(tmp_path / "tuned.safetensors", specs, 31)
    factors = write(tmp_path / "adapter.safetensors", pair("q", 192, 128, 6, DType.F32) + pair("down", 96, 320, 40, DType.F32), 32)
    pg = StubProcessGroup(1, 2)
    (l0, bufs), (l1, other), (l2, adapter) = (load(tmp_path / f"{n}.safetensors", pg=g) for n, g in
                                              (("base", pg), ("tuned", SingleGroup()), ("adapter", SingleGroup())))
    bufs.auto_mem_delete = False
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        bufs.merge_checkpoints([other], scale=1.0)
        bufs.merge_adapter(adapter, scale=2.0)
        with_adapter = {n: bufs.get_sharded(n, 0).clone() for n in shapes}
        bufs.merge_adapter(adapter, scale=-2.0)
        without = {n: bufs.get_sharded(n, 1).clone() for n in shapes}
    stream.synchronize()
    for n, (rows, cols) in shapes.items():
        w = base[n].double()
        o, s = polar(tuned[n].double() - w)
        a, b = (factors[f"{PREFIX}{n[:-7]}.lora_{k}.weight"].double() for k in "AB")
        merged, r = w + s * o, a.shape[0]
        # the orthogonal part as in the test above; each merge adds its own 32-bit roundings (six products per k, see close())
        slack = 1e-3 * s + (2 * (b.abs() @ a.abs()) * ((6 * r + 4) * 2.0**-23) + 2.0**-22 * (merged.abs() + 2 * (b @ a).abs())) * 2
        want, half = merged + 2 * (b @ a), rows // 2
        assert ((with_adapter[n].cpu().double() - want[half:]).abs() <= slack[half:]).all(), n
        assert ((without[n].cpu().double() - merged[:, cols // 2 :]).abs() <= slack[:, cols // 2 :]).all(), n
    for x in (bufs, other, adapter, l0, l1, l2):
        x.close()
