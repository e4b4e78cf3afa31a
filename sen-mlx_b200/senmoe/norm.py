"""RMS norm with the residual's addition, in 16 bits, in 8 bits with scales or
both, and its gradients: the step before the block,
``h = x + residual; y = norm(h)`` (deepseek_v2.rs:613-620), in one launch.

Sums are fp32 and each output is rounded once.  Nothing synchronises with the
host, so the calls can be captured into a CUDA graph, and nothing is recorded
for autograd.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import SenMoeNorm, SenMoeNormGrad, _check, lib
from .products import _CODES, _DTYPES, _bad, _current_stream, _rows
from .products8 import Rows8, _blocks, _device_of, _empty8, _like, _on16

_FIELD = {**_CODES, C.c_float: "f"}
_pack_norm = struct.Struct("".join(_FIELD[t] for _, t in SenMoeNorm._fields_)).pack
_pack_grad = struct.Struct("".join(_FIELD[t] for _, t in SenMoeNormGrad._fields_)).pack


class Normed(NamedTuple):
    """What ``rms_norm`` returns: y in 16 bits and in 8 (None where not asked
    for), and h, what was normed (x itself without a residual)."""
    y: torch.Tensor | None
    y8: Rows8 | None
    h: torch.Tensor


_F32 = torch.float32
_c_norm = None  # the library's entry, once it is loaded


def _operands(first: torch.Tensor, name: str, weight: torch.Tensor):
    """(dtype code, device, whether weight is fp32, row length)"""
    dtype, shape = first.dtype, first.shape
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{name} must be bfloat16 or float16, got {dtype}")
    device = _device_of(first)
    if not shape or shape[-1] < 1:
        raise _bad(f"{name} {tuple(shape)}")
    fp32 = weight.dtype is _F32
    if not fp32 and weight.dtype is not dtype or weight.get_device() != device:
        raise TypeError(f"weight must be {dtype} or float32 on cuda:{device}, got {weight.dtype} on {weight.device}")
    if weight.shape != shape[-1:]:
        raise _bad(f"weight {tuple(weight.shape)} for {name} {tuple(shape)}")
    return code, device, int(fp32), shape[-1]


def _same_rows(t: torch.Tensor, first: torch.Tensor, device: int, name: str):
    _on16(t, device, first.dtype, name)
    if t.shape != first.shape:
        raise _bad(f"{name} {tuple(t.shape)}, the rows are {tuple(first.shape)}")
    n = first.shape[-1]
    return (t, n) if t.is_contiguous() else _rows(t, n)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
             unit_offset: bool = False, sixteen_bit: bool = True, eight_bit: bool = False, stream=None) -> Normed:
    """h = x + residual (rounded to x's type), y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    x [..., n] bf16 or fp16, residual the same; weight [n] of x's type or fp32
    (``unit_offset``: 1 + weight).  ``eight_bit`` gives y as Rows8 (n a multiple
    of 32), ``sixteen_bit`` in x's type.
    """
    if stream is not None:
        with torch.cuda.stream(stream):
            return rms_norm(x, weight, eps, residual, unit_offset, sixteen_bit, eight_bit)
    code, device, fp32, n = _operands(x, "x", weight)
    if not sixteen_bit and not eight_bit:
        raise _bad("rms_norm: neither sixteen_bit nor eight_bit")
    nb = _blocks(n, "8-bit output: row length") if eight_bit else 0
    h, xs = (x, n) if x.is_contiguous() else _rows(x, n)
    ph = pr = rs = py = pc = ps = 0
    px, out_h = h.data_ptr(), x
    if residual is not None:
        residual, rs = _same_rows(residual, x, device, "residual")
        out_h = _like(x)
        pr, ph = residual.data_ptr(), out_h.data_ptr()
    if not weight.is_contiguous():
        weight = weight.contiguous()
    y = y8 = None
    if sixteen_bit:
        y = _like(x)
        py = y.data_ptr()
    if eight_bit:
        y8 = _empty8(x, x.shape[:-1], n)
        pc, ps = y8[0].data_ptr(), y8[1].data_ptr()
    global _c_norm
    if _c_norm is None:
        _c_norm = lib().senmoe_rms_norm
    status = _c_norm(
        _pack_norm(code, fp32, int(unit_offset), eps, x.numel() // n, n, px, xs, pr, rs, weight.data_ptr(), ph, n,
                   py, n, pc, n, ps, nb), _current_stream(device))
    if status:
        _check(status)
    return Normed(y, y8, out_h)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                      dh: torch.Tensor | None = None, unit_offset: bool = False, need_dx: bool = True,
                      need_dweight: bool = True, stream=None):
    """(dx, dweight) of ``rms_norm`` from dy [..., n] and its h; None where not
    needed.  ``dh`` is the gradient that reaches h beside the norm; with it, dx
    is the whole gradient of x and of the residual.  dweight has weight's type."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return rms_norm_backward(dy, h, weight, eps, dh, unit_offset, need_dx, need_dweight)
    code, device, fp32, n = _operands(h, "h", weight)
    rows = h.numel() // n
    dy, ys = _same_rows(dy, h, device, "dy")
    pd = ds = 0
    if dh is not None:
        dh, ds = _same_rows(dh, h, device, "dh")
        pd = dh.data_ptr()
    dx = _like(h) if need_dx else None
    h, hs = (h, n) if h.is_contiguous() else _rows(h, n)
    weight = weight.contiguous()
    dw = torch.empty_like(weight) if need_dweight else None
    args = (code, fp32, int(unit_offset), eps, rows, n, dy.data_ptr(), ys, h.data_ptr(), hs, weight.data_ptr(), pd, ds,
            dx.data_ptr() if need_dx else 0, n, dw.data_ptr() if need_dweight else 0)
    L, pws, need = lib(), 0, 0
    if need_dweight:
        need = L.senmoe_rms_norm_backward_workspace(_pack_grad(*args, 0, 0))
        if need < 0:
            _check(-need)
        if need:
            workspace = h.new_empty(need, dtype=torch.uint8)
            pws = workspace.data_ptr()
    status = L.senmoe_rms_norm_backward(_pack_grad(*args, pws, need), _current_stream(device))
    if status:
        _check(status)
    return dx, dw
