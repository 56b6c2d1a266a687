# SPDX-License-Identifier: Apache-2.0
"""Measured cases of the operators that change loaded weights.

``low_rank``       W' = W + scale * (up @ down) for the weights of one call, as an adapter file is merged into
                   a checkpoint (``merge_low_rank``).  Weights are fp32, bf16, fp16 or fp8 e4m3 with their
                   ``weight_scale``; the base weights stay and the merged ones go to buffers the caller keeps
                   (a server that swaps adapters).
``orthogonalize``  the nearest orthogonal matrix of an update by Newton-Schulz products (``orthogonalize``),
                   for one matrix or for the matrices of several layers in one call.

``run`` computes the plain form (elementary torch operations in 32 bits) or, with ``own``, makes the calls of the
package.  Shapes are those of the five benchmark checkpoints (``fastsafetensors_amd/checkpoints.py``).
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}

# (a, b, c) of each step of the iteration X <- aX + (bA + cA^2)X, A = XX^T
STEPS = [(3.4445, -4.7750, 2.0315)] * 5
EPS = 1e-7


def low_rank(name, shapes, rank, weights, factors, scale, layout="dense"):
    return {"name": name, "op": "low_rank", "shapes": shapes, "rank": rank, "weights": weights, "factors": factors,
            "scale": scale, "layout": layout}


def update(name, shapes, dtype, spectrum):
    return {"name": name, "op": "orthogonalize", "shapes": shapes, "dtype": dtype, "spectrum": spectrum}


def listed():
    # shapes travel as text ("768x2304 768x768"): a case is a dict of plain values
    return [
        # one projection of the GPT-2-small checkpoint, weights stored [in, out]: the smallest call, latency counts
        low_rank("gpt2s_attn_f32_r8", "768x2304", 8, "f32", "f32", 4.0, "in_out"),
        # three matrices of a GPT-2-medium layer, fp16, stored [in, out]
        low_rank("gpt2m_layer_f16_r16", "1024x1024 1024x4096 4096x1024", 16,
                 "f16", "f16", 2.0, "in_out"),
        # the seven matrices of a Llama-3-8B layer, a large adapter in bf16
        low_rank("llama8b_layer_bf16_r64", "4096x4096 1024x4096 1024x4096 4096x4096 14336x4096 14336x4096 4096x14336",
                 64, "bf16", "bf16", 0.5),
        # one rank's columns of a Llama-2-13B down projection, merged where they lie in the whole tensor; fp32 factors
        low_rank("llama13b_down_cut_bf16_r256", "5120x3456", 256, "bf16", "f32", 0.25, "pitched"),
        # the seven matrices of a Llama-3-70B fp8 layer
        low_rank("llama70b_layer_e4m3_r16", "8192x8192 1024x8192 1024x8192 8192x8192 28672x8192 28672x8192 8192x28672",
                 16, "e4m3", "bf16", 2.0),
        # odd widths and ranks: the embedding of GPT-2-small and a few ragged pieces
        low_rank("ragged_bf16_r5", "50257x767 1x4095 511x1 129x1025", 5, "bf16", "bf16", 1.5),
        # one projection's update, fp32 master weights
        update("gpt2s_attn_f32", "768x2304", "f32", "decaying"),
        # the output projections of all twelve layers in one call
        update("gpt2s_proj_x12_bf16", " ".join(["768x768"] * 12), "bf16", "flat"),
        # a key projection of the Llama-3-8B checkpoint
        update("llama8b_key_bf16", "1024x4096", "bf16", "decaying"),
        # its query projection, fp32
        update("llama8b_query_f32", "4096x4096", "f32", "spiked"),
        # its gate projection, taller than wide: the largest
        update("llama8b_gate_bf16", "14336x4096", "bf16", "decaying"),
        # odd sizes of several matrices, fp16, one of a single row
        update("ragged_f16", "1023x257 130x999 1x513 77x77", "f16", "flat"),
    ]


def spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        weights = rng.choice(["f32", "bf16", "bf16", "f16", "e4m3"])
        factors = rng.choice(["f32", "bf16", "f16"])
        left, shapes = 250_000_000, []
        for _ in range(rng.choice([1, 1, 2, 4, 7])):
            m, n = spread(rng, 1, 32768), spread(rng, 1, 32768)
            if m * n > left:
                n = max(1, left // m)
            left = max(1, left - m * n)
            shapes.append(f"{m}x{n}")
        case = low_rank("", " ".join(shapes), spread(rng, 1, 256), weights, factors, rng.choice([0.25, 0.5, 1.0, 1.7, 2.0, 8.0]),
                        rng.choice(["dense", "dense", "in_out", "pitched"]))
    else:
        left, shapes = 2.4e11, []
        for _ in range(rng.choice([1, 1, 1, 2, 5])):
            m, n = spread(rng, 1, 6000), spread(rng, 1, 6000)
            if min(m, n) ** 2 * max(m, n) > left:
                m = spread(rng, 1, 64)
            left -= min(m, n) ** 2 * max(m, n)
            shapes.append(f"{m}x{n}")
        case = update("", " ".join(shapes), rng.choice(["f32", "bf16", "f16"]), rng.choice(["flat", "decaying", "spiked"]))
    del case["name"]
    return case


def sizes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "low_rank":
        items, r = [], case["rank"]
        wt, ft = TYPES[case["weights"]], TYPES[case["factors"]]
        for m, n in sizes(case):
            # weights as a checkpoint holds them (normal, 0.02), the input factor as adapters begin (uniform within
            # 1/sqrt(in)), the output factor as training leaves it
            w, ws = normal(gen, m, n) * 0.02, None
            if case["weights"] == "e4m3":
                ws = torch.full((), 0.02 / 100.0, device="cuda")
                w = (w / ws).clamp_(-448.0, 448.0)
            w = w.to(wt)
            if case["layout"] == "pitched":  # columns of a tensor four times as wide
                whole = torch.empty((m, 4 * n), dtype=wt, device="cuda")
                whole[:, n : 2 * n].copy_(w)
                w = whole[:, n : 2 * n]
            fan_in, fan_out = (m, n) if case["layout"] == "in_out" else (n, m)
            lora_a = ((torch.rand((r, fan_in), generator=gen, device="cuda") * 2 - 1) / math.sqrt(fan_in)).to(ft)
            lora_b = (normal(gen, fan_out, r) * 0.01).to(ft)
            up, down = (lora_a.t(), lora_b.t()) if case["layout"] == "in_out" else (lora_b, lora_a)
            items.append((w, up, down, ws, torch.empty((m, n), dtype=wt, device="cuda")))
        return {"case": case, "items": items}
    mats = []
    for m, n in sizes(case):
        # momentum of a weight's gradient: a few strong directions over a floor of noise
        p = min(m, n)
        k = min(p, 32)
        left, right = normal(gen, m, k) / math.sqrt(m), normal(gen, k, n) / math.sqrt(n)
        if case["spectrum"] == "decaying":
            strength = 1.0 / torch.arange(1, k + 1, device="cuda")
        else:
            strength = torch.full((k,), 1.0 if case["spectrum"] == "spiked" else 0.0, device="cuda")
        floor = {"flat": 1.0, "decaying": 0.05, "spiked": 0.01}[case["spectrum"]]
        noise = normal(gen, m, n) / (math.sqrt(m) + math.sqrt(n))
        mats.append((((left * strength) @ right + floor * noise) * 1e-3).to(TYPES[case["dtype"]]))
    return {"case": case, "mats": mats}


def plain_low_rank(items, scale):
    outs = []
    for w, up, down, ws, _ in items:
        w32 = w.to(torch.float32)
        if ws is not None:
            w32 = w32 * ws
        merged = w32 + scale * (up.to(torch.float32) @ down.to(torch.float32))
        if ws is not None:
            merged = (merged / ws).clamp(-448.0, 448.0)
        outs.append(merged.to(w.dtype))
    return outs


def plain_orthogonalize(mats):
    outs = []
    for g in mats:
        x = g.to(torch.float32)
        tall = x.shape[0] > x.shape[1]
        if tall:
            x = x.t()
        x = x / (torch.sqrt((x * x).sum()) + EPS)
        for a, b, c in STEPS:
            gram = x @ x.t()
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        outs.append((x.t() if tall else x).to(g.dtype).contiguous())
    return outs


def run(state):
    case = state["case"]
    if case["op"] == "low_rank":
        if not own:
            return plain_low_rank(state["items"], case["scale"])
        from fastsafetensors_amd import LowRankUpdate, merge_low_rank

        return merge_low_rank([LowRankUpdate(w, up, down, case["scale"], weight_scale=ws, out=out)
                               for w, up, down, ws, out in state["items"]])
    if not own:
        return plain_orthogonalize(state["mats"])
    from fastsafetensors_amd import orthogonalize

    return orthogonalize(state["mats"], coefficients=STEPS, eps=EPS)


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits."""
    state = prepare(case, seed)
    outs = []
    if case["op"] == "low_rank":
        for w, up, down, ws, _ in state["items"]:
            merged = torch.matmul(up.double().contiguous(), down.double().contiguous()).mul_(case["scale"])
            held = 1.0 if ws is None else ws.double()
            merged = merged.div_(held).add_(w.double())
            outs.append(merged if ws is None else merged.clamp_(-448.0, 448.0))
        return outs
    if sum(min(s) * min(s) * max(s) for s in sizes(case)) > 3e11:
        return None
    for g in state["mats"]:
        # the polynomial acts on the singular values alone: x -> (aI + bS + cS^2) x for the Gram matrix S of the
        # smaller side, in whichever order the sides stand
        x = g.double()
        x = x / (x.square().sum().sqrt() + EPS)
        wide = x.shape[0] <= x.shape[1]
        for a, b, c in STEPS:
            if wide:
                s = torch.matmul(x, x.t().contiguous())
                poly = c * torch.matmul(s, s) + b * s
                poly.diagonal().add_(a)
                x = torch.matmul(poly, x)
            else:
                s = torch.matmul(x.t().contiguous(), x)
                poly = c * torch.matmul(s, s) + b * s
                poly.diagonal().add_(a)
                x = torch.matmul(x, poly)
        outs.append(x)
    return outs


def work(case):
    nbytes, flops = 0, 0
    for m, n in sizes(case):
        if case["op"] == "low_rank":
            r = case["rank"]
            nbytes += 2 * m * n * SIZE[case["weights"]] + (m + n) * r * SIZE[case["factors"]]
            flops += 2 * m * n * r
        else:
            p, q = min(m, n), max(m, n)
            nbytes += 2 * m * n * SIZE[case["dtype"]]
            # XX^T and A^2 are symmetric: half of each product
            flops += len(STEPS) * (p * p * q + p * p * p + 2 * p * p * q)
    return {"bytes": nbytes, "flops": flops}
