# SPDX-License-Identifier: Apache-2.0
"""Kernels that change weights in HBM, on torch tensors.

The reference only moves weights (its users merge adapters with the framework's own products);
here the merge runs as a streaming pass over the loaded weights.  ``merge_low_rank`` is what
``FilesBufferOnDevice.merge_adapter`` calls; it takes any tensors on the GPU.
"""

from dataclasses import dataclass
from typing import Any, List, Optional, Sequence, Tuple

import torch

from . import _native

_WEIGHT_TYPES = {
    torch.float32: _native.ELEM_TYPES["F32"],
    torch.float16: _native.ELEM_TYPES["F16"],
    torch.bfloat16: _native.ELEM_TYPES["BF16"],
    torch.float8_e4m3fn: _native.ELEM_TYPES["F8_E4M3"],
}
_FACTOR_TYPES = {t: n for t, n in _WEIGHT_TYPES.items() if t != torch.float8_e4m3fn}

# Workspace one library call is given at most when there are several updates: more are cut into
# several calls, so that an adapter for a whole checkpoint does not need its packed factors at once.
_WORKSPACE_BYTES = 512 * 1024 * 1024


@dataclass(eq=False)
class LowRankUpdate:
    """``weight + scale * (up @ down)``: ``weight`` [M, N] (fp32, fp16, bf16, or fp8 e4m3 with
    ``weight_scale``), ``up`` [M, r] and ``down`` [r, N] (fp32, fp16 or bf16, any strides).

    The result goes to ``out`` (a tensor of the weight's shape and type) or, without one, into
    ``weight`` itself.  ``weight`` and ``out`` have contiguous rows or contiguous columns, any
    distance apart.  ``weight_scale``: fp32, one value or one per row; the weight stands for
    ``weight * weight_scale`` and the result is requantised to the same scale, saturated to +-448."""

    weight: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor
    scale: float = 1.0
    weight_scale: Optional[torch.Tensor] = None
    out: Optional[torch.Tensor] = None


def _on_gpu(t: Any, what: str, device: Optional[torch.device], grad: bool) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor, not {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be in GPU memory (no CPU path exists)")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, the others are on {device}")
    if t.layout is not torch.strided:
        raise ValueError(f"{what} must be a dense tensor")
    if grad and t.requires_grad:
        raise RuntimeError(f"{what} requires a gradient, which this call does not provide: use torch.no_grad()")
    return t.device


def _by_rows(t: torch.Tensor) -> bool:
    return t.shape[1] <= 1 or t.stride(1) == 1


def _pitch(t: torch.Tensor, what: str) -> int:
    """Elements between rows of a matrix with contiguous rows."""
    m, n = t.shape
    if m <= 1:
        return n
    if t.stride(0) < n:
        raise ValueError(f"{what} with strides {tuple(t.stride())} has rows that overlap")
    return t.stride(0)


def _low_rank_desc(u: LowRankUpdate, device: Optional[torch.device], grad: bool) -> Tuple[torch.device, _native.FstxLowRankDesc]:
    w, up, down, ws = u.weight, u.up, u.down, u.weight_scale
    out = w if u.out is None else u.out
    device = _on_gpu(w, "weight", device, grad)
    _on_gpu(up, "up", device, grad)
    _on_gpu(down, "down", device, grad)
    if out is not w:
        _on_gpu(out, "out", device, grad)
    if w.dtype not in _WEIGHT_TYPES:
        raise TypeError(f"weight is {w.dtype}; fp32, fp16, bf16 and fp8 e4m3 are served")
    for t, what in ((up, "up"), (down, "down")):
        if t.dtype not in _FACTOR_TYPES:
            raise TypeError(f"{what} is {t.dtype}; fp32, fp16 and bf16 are served")
    if w.dim() != 2 or up.dim() != 2 or down.dim() != 2:
        raise ValueError("weight, up and down must have two dimensions")
    (m, n), r = w.shape, up.shape[1]
    if up.shape[0] != m or down.shape[0] != r or down.shape[1] != n:
        raise ValueError(f"shapes do not match: weight {tuple(w.shape)}, up {tuple(up.shape)}, down {tuple(down.shape)}")
    if out.shape != w.shape or out.dtype != w.dtype:
        raise ValueError(f"out is {tuple(out.shape)} {out.dtype}, weight {tuple(w.shape)} {w.dtype}")
    n_scales, ws_at = 0, None
    if w.dtype == torch.float8_e4m3fn:
        if ws is None:
            raise ValueError("an fp8 weight needs its weight_scale")
        _on_gpu(ws, "weight_scale", device, grad)
        if ws.dtype != torch.float32:
            raise TypeError(f"weight_scale is {ws.dtype}, not fp32")
        if not (ws.numel() == 1 or tuple(ws.shape) in ((m,), (m, 1))):
            raise ValueError(f"weight_scale {tuple(ws.shape)} is neither one value nor one per row of {tuple(w.shape)}")
        if not ws.is_contiguous():
            raise ValueError("weight_scale must be contiguous")
        n_scales, ws_at = ws.numel(), ws.data_ptr()
    elif ws is not None:
        raise ValueError(f"weight_scale goes with fp8 weights, not with {w.dtype}")
    if not (_by_rows(w) and _by_rows(out)):
        # stored by columns: the same merge of the transposed matrices
        w, out, up, down = w.t(), out.t(), down.t(), up.t()
        if not (_by_rows(w) and _by_rows(out)):
            raise ValueError("weight and out must both have contiguous rows, or both contiguous columns")
        if n_scales > 1:
            raise ValueError("a weight_scale per row needs a weight with contiguous rows")
    for t, what in ((up, "up"), (down, "down")):
        if min(t.stride()) < 0:
            raise ValueError(f"{what} has negative strides")
    return device, _native.FstxLowRankDesc(
        out.data_ptr(), w.data_ptr(), up.data_ptr(), down.data_ptr(), ws_at,
        w.shape[0], w.shape[1], r, _pitch(out, "out"), _pitch(w, "weight"),
        up.stride(0), up.stride(1), down.stride(0), down.stride(1),
        float(u.scale), _WEIGHT_TYPES[w.dtype], _FACTOR_TYPES[up.dtype], _FACTOR_TYPES[down.dtype], n_scales, 0,
    )


def _launch_low_rank(descs: Any, first: int, n: int, device: torch.device, need: int, stream: int) -> None:
    at = _native.ctypes.cast(_native.ctypes.byref(descs, first * _native.ctypes.sizeof(_native.FstxLowRankDesc)),
                             _native.ctypes.POINTER(_native.FstxLowRankDesc))
    if need < 0:
        need = _native.merge_low_rank_workspace(at, n)
    if need > _WORKSPACE_BYTES and n > 1:
        _launch_low_rank(descs, first, n // 2, device, -1, stream)
        _launch_low_rank(descs, first + n // 2, n - n // 2, device, -1, stream)
        return
    space = torch.empty(need, dtype=torch.uint8, device=device)
    _native.merge_low_rank(at, n, space.data_ptr() if need else 0, need, stream)


def merge_low_rank(updates: Sequence[LowRankUpdate]) -> List[torch.Tensor]:
    """Make every update's ``weight + scale * (up @ down)``; returns the tensors that hold the
    results (``out``, else ``weight``) in the order of ``updates``.

    All updates are checked before anything runs, and all of them leave as a few launches on the
    current stream of their device.  Products are summed in 32 bits and rounded once to the weight's
    type.  No result may overlap another result, another update's weight or a factor (that raises; column
    blocks of one tensor do not overlap).  There is no gradient: tensors that require one are refused
    while gradients are being recorded."""
    updates = list(updates)
    if not updates:
        return []
    grad = torch.is_grad_enabled()
    device: Optional[torch.device] = None
    descs = (_native.FstxLowRankDesc * len(updates))()
    for i, u in enumerate(updates):
        device, descs[i] = _low_rank_desc(u, device, grad)
    try:
        need = _native.merge_low_rank_workspace(descs, len(updates))
    except _native.NativeError as e:
        raise ValueError(f"merge_low_rank: results overlap what other updates read or write, or a size is out of range ({e})") from None
    outs = [u.weight if u.out is None else u.out for u in updates]
    with torch.cuda.device(device):
        _launch_low_rank(descs, 0, len(updates), device, need, torch.cuda.current_stream(device).cuda_stream)
    torch.autograd.graph.increment_version(outs)
    return outs
