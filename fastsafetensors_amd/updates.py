# SPDX-License-Identifier: Apache-2.0
"""Kernels that change weights in HBM, on torch tensors.

The reference only moves weights (its users merge adapters with the framework's own products);
here the merge runs as a streaming pass over the loaded weights.  ``merge_low_rank`` is what
``FilesBufferOnDevice.merge_adapter`` calls, ``orthogonalize`` -- the nearest orthogonal matrix of an
update -- what ``FilesBufferOnDevice.merge_checkpoints`` does; both take any tensors on the GPU.
"""

import contextlib
import math
import struct
from dataclasses import dataclass
from typing import Any, List, Optional, Sequence, Tuple, Union

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
    if t.is_neg():  # (the imaginary part of a conjugated tensor: its memory holds the other sign)
        raise ValueError(f"{what} is a negated view: give its resolve_neg()")
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


def _low_rank_desc(u: LowRankUpdate, device: torch.device, grad: bool) -> _native.FstxLowRankDesc:
    w, up, down, ws = u.weight, u.up, u.down, u.weight_scale
    out = w if u.out is None else u.out
    _on_gpu(w, "weight", device, grad)
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
    scale = float(u.scale)
    if not abs(scale) <= _LARGEST:
        raise ValueError(f"scale is {u.scale}, not a finite 32-bit number")
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
    return _native.FstxLowRankDesc(
        out.data_ptr(), w.data_ptr(), up.data_ptr(), down.data_ptr(), ws_at,
        w.shape[0], w.shape[1], r, _pitch(out, "out"), _pitch(w, "weight"),
        up.stride(0), up.stride(1), down.stride(0), down.stride(1),
        scale, _WEIGHT_TYPES[w.dtype], _FACTOR_TYPES[up.dtype], _FACTOR_TYPES[down.dtype], n_scales, 0,
    )


_DESC = struct.Struct("=14Qf5I")  # fstx_low_rank_desc
assert _DESC.size == _native.ctypes.sizeof(_native.FstxLowRankDesc)
_LARGEST = torch.finfo(torch.float32).max
_E4M3 = _WEIGHT_TYPES[torch.float8_e4m3fn]


def _pack_plain(buf: bytearray, at: int, u: LowRankUpdate, device: torch.device, grad: bool) -> bool:
    """Write the descriptor of an update with nothing unusual about it; False where ``_low_rank_desc`` has to look (and
    to say what is wrong).  A call costs a few microseconds per update on the host, as much as a small merge on the GPU."""
    w, up, down, ws, out, scale = u.weight, u.up, u.down, u.weight_scale, u.out, u.scale
    try:
        if out is None:
            out = w
        elif out.dtype is not w.dtype or out.shape != w.shape or out.device != device or (grad and out.requires_grad):
            return False
        wt, ut, dt = _WEIGHT_TYPES[w.dtype], _FACTOR_TYPES[up.dtype], _FACTOR_TYPES[down.dtype]
        (m, n), (m2, r), (r2, n2) = w.shape, up.shape, down.shape
        (src_pitch, one), (dst_pitch, out_one) = w.stride(), out.stride()
        if (
            not -_LARGEST <= scale <= _LARGEST or m != m2 or n != n2 or r != r2 or one != 1 or out_one != 1 or src_pitch < n or dst_pitch < n
            or w.device != device or up.device != device or down.device != device
            or (grad and (w.requires_grad or up.requires_grad or down.requires_grad))
            or w.is_neg() or up.is_neg() or down.is_neg() or out.is_neg() or (ws is not None and ws.is_neg())
        ):
            return False
        if wt == _E4M3:
            if ws is None or ws.numel() != 1 or ws.dtype is not torch.float32 or ws.device != device or (grad and ws.requires_grad):
                return False
            ws_at, n_scales = ws.data_ptr(), 1
        elif ws is not None:
            return False
        else:
            ws_at, n_scales = 0, 0
        _DESC.pack_into(buf, at, out.data_ptr(), w.data_ptr(), up.data_ptr(), down.data_ptr(), ws_at, m, n, r, dst_pitch, src_pitch,
                        *up.stride(), *down.stride(), scale, wt, ut, dt, n_scales, 0)
        return True
    except (AttributeError, KeyError, TypeError, ValueError, RuntimeError, struct.error):
        return False


def _low_rank_calls(descs: Any, first: int, n: int, need: int) -> List[Tuple[Any, int, int]]:
    """The library calls that ``descs`` are cut into: where they begin, how many, their workspace."""
    at = descs if first == 0 else _native.ctypes.cast(
        _native.ctypes.byref(descs, first * _DESC.size), _native.ctypes.POINTER(_native.FstxLowRankDesc))
    if need < 0:
        need = _native.merge_low_rank_workspace(at, n)
    if need > _WORKSPACE_BYTES and n > 1:
        return _low_rank_calls(descs, first, n // 2, -1) + _low_rank_calls(descs, first + n // 2, n - n // 2, -1)
    return [(at, n, need)]


def _launch_low_rank(descs: Any, n: int, device: torch.device, need: int, stream: int) -> None:
    calls = _low_rank_calls(descs, 0, n, need)
    # one workspace for all of them, which follow each other on the stream: if there is no memory for it, nothing has changed
    most = max(c[2] for c in calls)
    space = torch.empty(most, dtype=torch.uint8, device=device) if most else None
    for at, count, bytes_ in calls:
        _native.merge_low_rank(at, count, 0 if space is None else space.data_ptr(), bytes_, stream)


def _on_device(device: torch.device) -> Any:
    """Makes ``device`` the current one where it is not (the kernels are launched on the current device)."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


_HERE = contextlib.nullcontext()


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
    grad, n = torch.is_grad_enabled(), len(updates)
    device = _on_gpu(updates[0].weight, "weight", None, False)
    buf = bytearray(n * _DESC.size)
    descs = (_native.FstxLowRankDesc * n).from_buffer(buf)
    for i, u in enumerate(updates):
        if not _pack_plain(buf, i * _DESC.size, u, device, grad):
            descs[i] = _low_rank_desc(u, device, grad)
    try:
        need = _native.merge_low_rank_workspace(descs, n)
    except _native.NativeError as e:
        raise ValueError(f"merge_low_rank: results overlap what other updates read or write, or a size is out of range ({e})") from None
    outs = [u.weight if u.out is None else u.out for u in updates]
    with _on_device(device):
        _launch_low_rank(descs, n, device, need, torch.cuda.current_stream(device).cuda_stream)
    torch.autograd.graph.increment_version(outs)
    return outs


# a, b, c of five steps that take singular values from 0.0015 of |G|_F up into 0.68 .. 1.21, with a slope at zero that
# comes at the price of not ending at 1; 0.001 of |G|_F ends at 0.47, smaller ones at up to 485 times themselves
DEFAULT_COEFFICIENTS = ((3.4445, -4.7750, 2.0315),) * 5

# ... followed by steps with a fixed point of third order at 1: singular values from 0.0005 of |G|_F up end within 3e-4 of 1,
# from 0.0007 within 1e-6
POLAR_COEFFICIENTS = DEFAULT_COEFFICIENTS + ((1.875, -1.25, 0.375),) * 4


# sides that fstx_orthogonalize takes: the longer and the shorter one
MAX_SIDE, MAX_SHORT_SIDE = 1 << 20, 1 << 16


def orthogonalize(
    updates: Union[torch.Tensor, Sequence[torch.Tensor]],
    coefficients: Sequence[Sequence[float]] = DEFAULT_COEFFICIENTS,
    eps: float = 1e-7,
    outs: Optional[Sequence[torch.Tensor]] = None,
) -> Union[torch.Tensor, List[torch.Tensor]]:
    """The nearest orthogonal matrix of every update (fp32, fp16 or bf16, two dimensions, any strides,
    up to 2^20 a side, the shorter one up to 2^16) approximated by Newton-Schulz steps on ``X = G / (|G|_F + eps)``: for each ``(a, b, c)``
    ``X <- a X + (b A + c A^2) X`` with ``A = X X^T`` (the shorter side as rows).

    Returns new tensors of the updates' shapes and types, or fills ``outs`` (contiguous rows or
    contiguous columns; an update may be its own ``out``, but not overlap it partly).  One tensor in, one tensor out; a sequence gives a list.
    The matrices of one call run together, so that small ones share launches.  All are checked before
    anything runs.  The iterates and the operands of all products are held in 22 bits, sums in 32, whatever the
    update's type; the result is rounded to it once.  Updates far smaller than ``eps`` keep these bits.

    Up to 32 rows or columns everything is done in 64 bits.  Coefficients and eps are taken as 32-bit numbers.  A call takes 12 bytes of workspace per element of its matrices and
    8 per element of their squares, up to 4 GiB and more only for a matrix that alone needs more.

    The default coefficients take singular values from 0.0015 of the update's Frobenius norm up into 0.68 to 1.21, which is
    what an optimiser needs; ``POLAR_COEFFICIENTS`` takes them to 1 (from 0.0005 of the norm up, within 3e-4).  Smaller ones are
    multiplied by up to 485, or 6000, and stay small.  Coefficients must keep the
    iterates' singular values at 2 or less.  There is no gradient: tensors that require one are refused while
    gradients are being recorded."""
    single = isinstance(updates, torch.Tensor)
    if outs is not None:
        outs = [outs] if single and isinstance(outs, torch.Tensor) else list(outs)
    call = Orthogonalization([updates] if single else list(updates), coefficients, eps, outs)
    if call.device is not None:
        call.launch(torch.empty(call.need, dtype=torch.uint8, device=call.device))
        if outs is not None:
            torch.autograd.graph.increment_version(outs)
    return call.outs[0] if single else call.outs


class Orthogonalization:
    """A checked call of ``orthogonalize``: ``need`` bytes of workspace, then ``launch``."""

    def __init__(
        self,
        mats: List[torch.Tensor],
        coefficients: Sequence[Sequence[float]],
        eps: float,
        outs: Optional[List[torch.Tensor]],
    ) -> None:
        flat = [float(v) for step in coefficients for v in step]
        if not all(len(step) == 3 for step in coefficients) or not 1 <= len(flat) // 3 <= 64:
            raise ValueError("coefficients must be 1 to 64 triples (a, b, c)")
        if not all(math.isfinite(v) for v in flat) or not (math.isfinite(eps) and eps >= 0):
            raise ValueError("coefficients must be finite, eps finite and not negative")
        if not all(abs(v) <= _LARGEST for v in (*flat, eps)):
            raise ValueError("coefficients and eps must be 32-bit numbers")
        if outs is not None and len(outs) != len(mats):
            raise ValueError(f"{len(outs)} outs for {len(mats)} updates")
        grad = torch.is_grad_enabled()
        device: Optional[torch.device] = None
        for i, g in enumerate(mats):
            device = _on_gpu(g, "update", device, grad)
            if g.dtype not in _FACTOR_TYPES:
                raise TypeError(f"update is {g.dtype}; fp32, fp16 and bf16 are served")
            if g.dim() != 2:
                raise ValueError(f"update {tuple(g.shape)} does not have two dimensions")
            if outs is not None:
                _on_gpu(outs[i], "out", device, grad)
                if outs[i].shape != g.shape or outs[i].dtype != g.dtype:
                    raise ValueError(f"out is {tuple(outs[i].shape)} {outs[i].dtype}, update {tuple(g.shape)} {g.dtype}")
        if outs is None:
            outs = [torch.empty(g.shape, dtype=g.dtype, device=device) for g in mats]
        descs = (_native.FstxOrthogonalizeDesc * len(mats))()
        for d, g, out in zip(descs, mats, outs):
            if not _by_rows(out):  # the transposed problem is the same one
                g, out = g.t(), out.t()
                if not _by_rows(out):
                    raise ValueError("out must have contiguous rows or contiguous columns")
            d.dst, d.src = out.data_ptr(), g.data_ptr()
            d.rows, d.cols = g.shape
            d.dst_pitch = _pitch(out, "out")
            d.src_row_stride, d.src_col_stride = g.stride()
            d.type = _FACTOR_TYPES[g.dtype]
        self.device, self.mats, self.outs, self.need = device, mats, outs, 0
        self._args = (descs, len(mats), (_native.ctypes.c_float * len(flat))(*flat), len(flat) // 3)
        self._eps = float(eps)
        if device is None:
            return
        with _on_device(device):
            try:
                self.need = _native.orthogonalize_workspace(*self._args)
            except _native.NativeError as e:
                raise ValueError(f"orthogonalize: outs overlap each other or other updates, or a size is out of range ({e})") from None

    def launch(self, space: torch.Tensor) -> None:
        """Queue the work on the current stream, with the first ``need`` bytes of ``space``."""
        with _on_device(self.device):
            _native.orthogonalize(*self._args, self._eps, space.data_ptr() if self.need else 0, self.need,
                                  torch.cuda.current_stream(self.device).cuda_stream)
