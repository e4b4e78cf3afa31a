"""Rows in 8 bits and the linear products over them.

``Rows8`` holds a matrix in e4m3 elements with a power-of-two scale (e8m0) for
every 32 of a row, the smallest with which the 32 are at most 448: an element
is off by half a step of three fraction bits.  ``rms_norm`` and the products
write such rows, ``quantize8`` makes them of 16-bit ones (weights, once).

* ``linear8(x, weight, ...)``: ``y = act(x @ weight.T + bias) + residual`` of
  the values the bytes stand for, as ``linear``, at twice its rate; ``y`` in 16
  bits, or with ``eight_bit`` in 8;
* ``grouped_linear8(x, weight, offsets, ...)``: one weight matrix per expert
  over rows in expert order, as ``grouped_linear``;
* ``linear8_input_grad`` / ``grouped_linear8_input_grad``: the gradient of x
  from dy, through the weight's transpose in 8 bits and dz in 8 bits.

A gated pair (``swiglu``, ``geglu``: weight holds the gate's rows, then the
up's) with ``eight_bit`` is the first half of a feed-forward block in one
launch; ``linear8`` over its rows is the second.  The weight's gradient is a
sum over rows, which the blocks of 32 do not follow: ``linear_backward`` and
``grouped_linear_backward`` with ``need_dx=False`` take it from 16-bit rows.

Sums are fp32 and each output is rounded once.  Nothing synchronises with the
host, so the calls can be captured into a CUDA graph; ``linear_check`` reports
waits that ran out.  They record nothing for autograd.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import ERR_UNSUPPORTED, SenMoeError, SenMoeLinear8, SenMoeQuantize8, _check, lib
from .products import (_CODES, _DTYPES, _GATED, ACTIVATIONS, LINEAR_AUTO, _bad, _current_device, _current_stream,
                       _no_activation, _rows)

BLOCK8 = 32  # elements of a scale
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_pack_quantize = struct.Struct("".join(_CODES[t] for _, t in SenMoeQuantize8._fields_)).pack
_c_quantize = _c_linear8 = None  # the library's entries, once it is loaded
_pack_linear8 = struct.Struct("".join(_CODES[t] for _, t in SenMoeLinear8._fields_)).pack


class Rows8(NamedTuple):
    """codes float8_e4m3fn [..., n] and scales float8_e8m0fnu [..., n / 32]."""
    codes: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values (exact in fp32 and bf16, but for magnitudes at the end of their range)."""
        v = self.codes.float().unflatten(-1, (-1, BLOCK8)) * self.scales.float()[..., None]
        return v.flatten(-2).to(dtype)

    def take(self, index: torch.Tensor) -> "Rows8":
        """The rows (of the first dimension) at ``index``."""
        return Rows8(self.codes.view(torch.uint8)[index].view(_E4M3), self.scales.view(torch.uint8)[index].view(_E8M0))


def _blocks(n: int, what: str) -> int:
    if n % BLOCK8 or n < 1:
        raise SenMoeError(ERR_UNSUPPORTED, f"{what} {n}: 8-bit rows are whole blocks of {BLOCK8}")
    return n // BLOCK8


def _check_rows8(r, name: str, device: int):
    """The shape of r's codes."""
    codes, scales = r
    if codes.dtype is not _E4M3 or scales.dtype is not _E8M0:
        raise TypeError(f"{name} must hold float8_e4m3fn codes and float8_e8m0fnu scales, got {codes.dtype} and "
                        f"{scales.dtype}")
    if codes.get_device() != device or scales.get_device() != device:
        raise TypeError(f"{name} on {codes.device} and {scales.device}: tensors must share one device")
    shape = codes.shape
    if not shape:
        raise _bad(f"{name} has no dimension")
    n = shape[-1]
    if n % BLOCK8 or n < 1:
        _blocks(n, f"{name}: row length")
    if scales.shape != (*shape[:-1], n // BLOCK8):
        raise _bad(f"{name}: scales {tuple(scales.shape)} for codes {tuple(shape)}")
    return shape


def _rows8(r, name: str) -> Rows8:
    if not isinstance(r, Rows8):
        raise TypeError(f"{name} must be Rows8, got {type(r).__name__}")
    return r


# A decode step's kernels take a few microseconds, and an allocation two or
# three on the host: empty_like and empty_strided are the cheapest forms of one.
def _like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _empty(t: torch.Tensor, lead, n: int, dtype) -> torch.Tensor:
    """An uninitialised contiguous [*lead, n] on t's device."""
    if len(lead) == 1:
        return torch.empty_strided((lead[0], n), (n, 1), dtype=dtype, device=t.device)
    return t.new_empty((*lead, n), dtype=dtype)


def _empty8(t: torch.Tensor, lead, n: int) -> Rows8:
    """Uninitialised rows of n elements on t's device."""
    return Rows8(_empty(t, lead, n, _E4M3), _empty(t, lead, n // BLOCK8, _E8M0))


def _device_of(t: torch.Tensor) -> int:
    device = t.get_device()
    if device < 0:
        raise TypeError("tensors must be CUDA tensors")
    if device != _current_device():
        raise _bad(f"tensors on {t.device}, current device is cuda:{_current_device()}")
    return device


def _flat8(r: Rows8, n: int):
    """(codes, their stride, scales, their stride) of rows the kernels can read; copies where a row is not."""
    codes, scales = r
    if codes.is_contiguous() and not codes.data_ptr() & 15 and not n & 15:
        cs = n
    else:
        codes, cs = _rows(codes, n)
        if (codes.data_ptr() | cs) & 15:
            codes, cs = codes.clone(memory_format=torch.contiguous_format), n
    b = n // BLOCK8
    if scales.is_contiguous():
        return codes, cs, scales, b
    return codes, cs, *_rows(scales, b)


def _stacked(t: torch.Tensor, n: int, k: int, grid: int):
    """t [n, k] or [E, n, k]: (t, row stride, group stride), copied where strides or base do not allow it."""
    s, grouped = t.stride(), t.dim() == 3
    ok = not (s[-1] != 1 and k > 1 or s[-2] < k and n > 1 or grouped and t.shape[0] > 1 and s[0] < (n - 1) * s[-2] + k)
    rs = s[-2] if n > 1 else k
    gs = s[0] if grouped and t.shape[0] > 1 else n * rs
    if ok and not (t.data_ptr() | rs | gs) % grid:
        return t, rs, gs
    return t.clone(memory_format=torch.contiguous_format), k, n * k


def _on16(t: torch.Tensor, device: int, dtype, name: str) -> None:
    if t.dtype is not dtype or t.get_device() != device:
        raise TypeError(f"{name} must be {dtype} on cuda:{device}, got {t.dtype} on {t.device}")


def quantize8(x: torch.Tensor, stream=None) -> Rows8:
    """x [..., n] (bf16 or fp16, n a multiple of 32) in 8 bits with scales."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return quantize8(x)
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    device = _device_of(x)
    if not x.dim():
        raise _bad("x has no dimension")
    return _quantize(x, None, 0, device)


def _quantize(x, preact, act: int, device: int) -> Rows8:
    """x, or dz = x act'(preact), in 8 bits."""
    n = x.shape[-1]
    _blocks(n, "row length")
    wide = 2 * n if act >= _GATED else n
    out = _empty8(x, x.shape[:-1], wide)
    _run_quantize(x, preact, act, n, wide, out[0].data_ptr(), out[1].data_ptr(), device)
    return out


def _run_quantize(x, preact, act, n, wide, codes, scales, device) -> None:
    xs, zs, pz = n, wide, 0
    if not x.is_contiguous():
        x, xs = _rows(x, n)
    if act:
        if not preact.is_contiguous():
            preact, zs = _rows(preact, wide)
        pz = preact.data_ptr()
    global _c_quantize
    if _c_quantize is None:
        _c_quantize = lib().senmoe_quantize8
    status = _c_quantize(
        _pack_quantize(_DTYPES[x.dtype], act, x.numel() // n, n, x.data_ptr(), xs, pz, zs, codes, wide, scales,
                       wide // BLOCK8), _current_stream(device))
    if status:
        _check(status)


def _run_linear8(*args, device) -> None:
    global _c_linear8
    if _c_linear8 is None:
        _c_linear8 = lib().senmoe_linear8
    status = _c_linear8(_pack_linear8(*args), _current_stream(device))
    if status:
        _check(status)


def _check_offsets(offsets: torch.Tensor, experts: int, device: int) -> None:
    if offsets.dtype is not torch.int32 or offsets.get_device() != device:
        raise TypeError(f"offsets must be int32 on cuda:{device}, got {offsets.dtype} on {offsets.device}")
    if offsets.dim() != 1 or offsets.shape[0] != experts + 1:
        raise _bad(f"offsets {tuple(offsets.shape)} for {experts} experts")


def _product8(x, weight, offsets, bias, residual, activation, save_preact, eight_bit, dtype, stream, path):
    if stream is not None:  # temporaries and outputs belong to the stream of the launch
        with torch.cuda.stream(stream):
            return _product8(x, weight, offsets, bias, residual, activation, save_preact, eight_bit, dtype, None, path)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise _no_activation(activation)
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    device = _device_of(_rows8(x, "x")[0])
    shape = _check_rows8(x, "x", device)
    wshape = _check_rows8(_rows8(weight, "weight"), "weight", device)
    if len(wshape) != (2 if offsets is None else 3):
        raise _bad(f"weight must be {'[out, in]' if offsets is None else '[experts, out, in]'}, got {tuple(wshape)}")
    wide, k = wshape[-2], wshape[-1]
    if shape[-1] != k:
        raise _bad(f"x {tuple(shape)} against weight {tuple(wshape)}")
    if wide < 1:
        raise _bad(f"weight {tuple(wshape)}: out_features={wide}")
    n = wide
    if act >= _GATED:
        if wide % 2:
            raise _bad(f"{activation}: weight has {wide} rows, gate and up need an even number")
        n = wide // 2
    groups = 1
    if offsets is not None:
        if len(shape) != 2:
            raise _bad(f"x must be [rows, in], got {tuple(shape)}")
        groups = wshape[0]
        _check_offsets(offsets, groups, device)
        offsets = offsets.contiguous()
    lead = shape[:-1]
    pb = pr = rs = py = ys = pc = ps = pz = 0
    if bias is not None:
        _on16(bias, device, dtype, "bias")
        if bias.numel() != groups * wide or not bias.dim() or bias.shape[-1] != wide:
            raise _bad(f"bias {tuple(bias.shape)} for weight {tuple(wshape)}")
        bias = bias.contiguous()
        pb = bias.data_ptr()
    if residual is not None:
        _on16(residual, device, dtype, "residual")
        if residual.shape != (*lead, n):
            raise _bad(f"residual {tuple(residual.shape)}, the output is {(*lead, n)}")
        residual, rs = (residual, n) if residual.is_contiguous() else _rows(residual, n)
        pr = residual.data_ptr()
    codes, xs, scales, ss = _flat8(x, k)
    w, ws, wg = _stacked(weight.codes, wide, k, 16)
    b = k // BLOCK8
    sw, sws, swg = _stacked(weight.scales, wide, b, 1)
    if eight_bit:
        nb = _blocks(n, "8-bit output: row length")
        out = _empty8(codes, lead, n)
        pc, ps = out[0].data_ptr(), out[1].data_ptr()
    else:
        nb = 0
        out = _empty(codes, lead, n, dtype)
        py = out.data_ptr()
    z = None
    if save_preact:
        z = _empty(codes, lead, wide, dtype)
        pz = z.data_ptr()
    rows = codes.numel() // k
    if rows:
        _run_linear8(code, act, groups, path, rows, k, n, codes.data_ptr(), xs, scales.data_ptr(), ss,
                     w.data_ptr(), ws, wg, sw.data_ptr(), sws, swg, 0 if offsets is None else offsets.data_ptr(), pb,
                     pr, rs, py, n, pc, n, ps, nb, pz, wide, device=device)
    return (out, z) if save_preact else out


def linear8(x: Rows8, weight: Rows8, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
            activation: str = "none", save_preact: bool = False, eight_bit: bool = False,
            dtype: torch.dtype = torch.bfloat16, stream=None, path: int = LINEAR_AUTO):
    """act(x [..., in] @ weight [wide, in].T + bias [wide]) + residual [..., out] -> [..., out].

    The output is ``dtype`` (that of bias, residual and pre-activations too), or
    Rows8 with ``eight_bit`` (out a multiple of 32).  ``save_preact`` also
    returns what the activation was applied to, [..., wide] in ``dtype``, for
    ``linear8_input_grad`` and ``linear_backward``.
    """
    return _product8(x, weight, None, bias, residual, activation, save_preact, eight_bit, dtype, stream, path)


def grouped_linear8(x: Rows8, weight: Rows8, offsets: torch.Tensor, bias: torch.Tensor | None = None,
                    activation: str = "none", save_preact: bool = False, eight_bit: bool = False,
                    dtype: torch.dtype = torch.bfloat16, stream=None, path: int = LINEAR_AUTO):
    """linear8 with weight [E, wide, in] and bias [E, wide] of each row's
    expert; x [S, in] in expert order, offsets int32 [E + 1].  Rows outside
    [offsets[0], offsets[E]) come out as zero."""
    if offsets is None:
        raise _bad("offsets is None")
    return _product8(x, weight, offsets, bias, None, activation, save_preact, eight_bit, dtype, stream, path)


def _input_grad(dy, weight_t, offsets, preact, activation, stream, path):
    if stream is not None:
        with torch.cuda.stream(stream):
            return _input_grad(dy, weight_t, offsets, preact, activation, None, path)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise _no_activation(activation)
    if dy.dtype not in _DTYPES:
        raise TypeError(f"dy must be bfloat16 or float16, got {dy.dtype}")
    device = _device_of(dy)
    if not dy.dim():
        raise _bad("dy has no dimension")
    wshape = _check_rows8(_rows8(weight_t, "weight_t"), "weight_t", device)
    n = dy.shape[-1]
    wide = 2 * n if act >= _GATED else n
    if wshape[-1] != wide:
        raise _bad(f"dy {tuple(dy.shape)} against weight_t {tuple(wshape)}")
    if act:
        if preact is None or preact.shape != (*dy.shape[:-1], wide):
            raise _bad(f"{activation}: preact {None if preact is None else tuple(preact.shape)}, "
                       f"{(*dy.shape[:-1], wide)} wanted")
        _on16(preact, device, dy.dtype, "preact")
    _blocks(n, "dy: row length")
    if len(wshape) != (2 if offsets is None else 3):
        raise _bad(f"weight_t must be {'[in, out]' if offsets is None else '[experts, in, out]'}, got {tuple(wshape)}")
    k = wshape[-2]
    if k < 1:
        raise _bad(f"weight_t {tuple(wshape)}: in_features={k}")
    groups = 1
    if offsets is not None:
        if dy.dim() != 2:
            raise _bad(f"dy must be [rows, out], got {tuple(dy.shape)}")
        groups = wshape[0]
        _check_offsets(offsets, groups, device)
        offsets = offsets.contiguous()
    rows, lead = dy.numel() // n, dy.shape[:-1]
    dx = _empty(dy, lead, k, dy.dtype)
    if rows:
        size = rows * wide  # dz: its elements, then its scales
        held = _empty(dy, (1,), size + size // BLOCK8, torch.uint8)  # (until both calls are made)
        dz = held.data_ptr()
        _run_quantize(dy, preact, act, n, wide, dz, dz + size, device)
        w, ws, wg = _stacked(weight_t.codes, k, wide, 16)
        sw, sws, swg = _stacked(weight_t.scales, k, wide // BLOCK8, 1)
        _run_linear8(_DTYPES[dy.dtype], 0, groups, path, rows, wide, k, dz, wide, dz + size, wide // BLOCK8,
                     w.data_ptr(), ws, wg, sw.data_ptr(), sws, swg, 0 if offsets is None else offsets.data_ptr(), 0,
                     0, 0, dx.data_ptr(), k, 0, 0, 0, 0, 0, 0, device=device)
    return dx


def linear8_input_grad(dy: torch.Tensor, weight_t: Rows8, preact: torch.Tensor | None = None,
                       activation: str = "none", stream=None, path: int = LINEAR_AUTO) -> torch.Tensor:
    """dx [..., in] of ``linear8`` from dy [..., out]: dz = dy act'(preact) in 8
    bits, times the weight.  ``weight_t`` is ``quantize8`` of its transpose, [in,
    wide]; ``preact`` is what ``save_preact`` returned."""
    return _input_grad(dy, weight_t, None, preact, activation, stream, path)


def grouped_linear8_input_grad(dy: torch.Tensor, weight_t: Rows8, offsets: torch.Tensor,
                               preact: torch.Tensor | None = None, activation: str = "none", stream=None,
                               path: int = LINEAR_AUTO) -> torch.Tensor:
    """dx [S, in] of ``grouped_linear8`` from dy [S, out]; weight_t [E, in, wide]."""
    if offsets is None:
        raise _bad("offsets is None")
    return _input_grad(dy, weight_t, offsets, preact, activation, stream, path)
