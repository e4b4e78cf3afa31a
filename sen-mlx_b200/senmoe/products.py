"""Linear products over 16-bit (bf16 or fp16) weights and their gradients.

* ``linear(x, weight, ...)``: ``y = act(x @ weight.T + bias) + residual``, the
  reference's ``nn::Linear::forward`` (deepseek_v2.rs:528) with the steps that
  follow it in the same launch;
* ``grouped_linear(x, weight, offsets, ...)``: the same with one weight matrix
  per expert over rows in expert order: row ``s`` takes ``weight[e]`` for
  ``offsets[e] <= s < offsets[e + 1]`` (``dispatch``'s offsets, or a slice of
  them for a rank's own experts);
* ``linear_backward`` / ``grouped_linear_backward``: the gradients of x, weight
  and bias (the residual's is ``dy``).

Activations: ``none``, ``relu``, ``silu``, ``gelu``, ``gelu_tanh``, and the
gated pairs ``swiglu`` (silu) and ``geglu`` (tanh gelu), whose weight, bias and
pre-activation hold ``2 * out`` rows, the gate's first.  Sums are fp32 and the
result is rounded once.  Nothing synchronises with the host, so the calls can
be captured into a CUDA graph.

The calls record nothing for autograd: what they return has no ``grad_fn``,
whatever their arguments require.  Training calls the ``_backward`` functions,
or wraps a pair in a ``torch.autograd.Function``.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import ERR_BAD_ARG, SenMoeError, SenMoeLinear, SenMoeLinearGrad, _check, lib

# SenMoeLinearPath
LINEAR_AUTO, LINEAR_ANY, LINEAR_TCGEN05, LINEAR_SMALL = 0, 1, 2, 3
LINEAR_TCGEN05_ONE, LINEAR_TCGEN05_PAIR, LINEAR_TCGEN05_SPLIT = 4, 5, 6
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5, "geglu": 6}
_GATED = 5  # from here on: gated pairs
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}

# A decode step's product takes a few microseconds on the GPU, so the calls
# keep their host side short: the argument structs are packed by one call
# (their layout is the ctypes mirror's) and the current stream is read as the
# handle that the C entry takes.
_CODES = {C.c_int32: "i", C.c_int64: "q", C.c_void_p: "P"}
_pack_linear = struct.Struct("".join(_CODES[t] for _, t in SenMoeLinear._fields_)).pack
_pack_grad = struct.Struct("".join(_CODES[t] for _, t in SenMoeLinearGrad._fields_)).pack
_c_linear = None  # the library's entry, once it is loaded
# (None in a torch without CUDA, which has no tensor that gets as far.)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _bad(message: str) -> SenMoeError:
    return SenMoeError(ERR_BAD_ARG, message)


def _rows(t: torch.Tensor, n: int) -> tuple[torch.Tensor, int]:
    """t [..., n] as (rows of n contiguous elements, their stride), a view where the strides allow one."""
    if t.dim() != 2:
        t = t.reshape(-1, n)
    s0, s1 = t.stride()
    if s1 != 1 and n > 1 or s0 < n and t.shape[0] > 1:
        return t.contiguous(), n
    return t, s0 if s0 > n else n


def _matrices(w: torch.Tensor, n: int, k: int) -> tuple[torch.Tensor, int, int]:
    """w [n, k] or [E, n, k]: (w, row stride, group stride)."""
    s = w.stride()
    if not (s[-1] != 1 and k > 1 or s[-2] < k and n > 1 or len(s) == 3 and w.shape[0] > 1 and s[0] < n * s[-2]):
        return w, s[-2] if s[-2] > k else k, s[0] if len(s) == 3 else 0
    return w.contiguous(), k, n * k


def _no_activation(name) -> SenMoeError:
    return _bad(f"activation {name!r}: one of {', '.join(ACTIVATIONS)}")


def _same(t: torch.Tensor, first: torch.Tensor, dtype, device: int) -> None:
    if t.dtype is not dtype or t.get_device() != device:
        raise TypeError(f"tensors must share one dtype and device: {dtype} on {first.device}, {t.dtype} on {t.device}")


def _operands(first: torch.Tensor, *others) -> tuple[int, int]:
    """(the common 16-bit dtype's code, the device): every tensor on the current CUDA device."""
    dtype, device = first.dtype, first.get_device()
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"tensors must be bfloat16 or float16, got {dtype}")
    if device < 0:
        raise TypeError("tensors must be CUDA tensors")
    for t in others:
        _same(t, first, dtype, device)
    if device != _current_device():
        raise _bad(f"tensors on {first.device}, current device is cuda:{_current_device()}")
    return code, device


def _check_groups(offsets: torch.Tensor, weight: torch.Tensor, x: torch.Tensor) -> None:
    if weight.dim() != 3:
        raise _bad(f"weight must be [experts, out, in], got {tuple(weight.shape)}")
    if offsets.dtype is not torch.int32 or offsets.get_device() != x.get_device():
        raise TypeError(f"offsets must be int32 on {x.device}, got {offsets.dtype} on {offsets.device}")
    if offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
        raise _bad(f"offsets {tuple(offsets.shape)} for {weight.shape[0]} experts")


def _forward(x, weight, offsets, bias, residual, activation, save_preact, stream, out, path):
    if stream is not None:  # temporaries and outputs belong to the stream of the launch
        with torch.cuda.stream(stream):
            return _forward(x, weight, offsets, bias, residual, activation, save_preact, None, out, path)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise _no_activation(activation)
    code, device = _operands(x, weight)
    wshape, shape = weight.shape, x.shape
    wide, k = wshape[-2], wshape[-1]
    if not shape or shape[-1] != k:
        raise _bad(f"x {tuple(shape)} against weight {tuple(wshape)}")
    if wide < 1 or k < 1:
        raise _bad(f"weight {tuple(wshape)}: in_features={k} out_features={wide}")
    n = wide
    if act >= _GATED:
        if wide % 2:
            raise _bad(f"{activation}: weight has {wide} rows, gate and up need an even number")
        n = wide // 2
    groups = 1
    if offsets is not None:
        groups, offsets = wshape[0], offsets.contiguous()
    pb = pr = pz = rs = 0
    if bias is not None:
        _same(bias, x, x.dtype, device)
        if bias.numel() != groups * wide or not bias.dim() or bias.shape[-1] != wide:
            raise _bad(f"bias {tuple(bias.shape)} for weight {tuple(wshape)}")
        bias = bias if bias.is_contiguous() else bias.contiguous()
        pb = bias.data_ptr()
    lead = shape[:-1]
    shape = (*lead, n)
    if residual is not None:
        _same(residual, x, x.dtype, device)
        if residual.shape != shape:
            raise _bad(f"residual {tuple(residual.shape)}, the output is {shape}")
        rs = n
        if not residual.is_contiguous():
            residual, rs = _rows(residual, n)
        pr = residual.data_ptr()
    xs = ws = k
    gs = wide * k
    if not x.is_contiguous():
        x, xs = _rows(x, k)
    if not weight.is_contiguous():
        weight, ws, gs = _matrices(weight, wide, k)
    rows = x.numel() // k
    if out is None:
        out = y = x.new_empty(shape)
        ys = n
    else:
        _same(out, x, x.dtype, device)
        if out.shape != shape or n > 1 and out.stride(-1) != 1:
            raise _bad(f"out {tuple(out.shape)} strides {out.stride()}, the output is {shape}, its rows contiguous")
        try:
            y = out if out.dim() == 2 else out.view(-1, n)
        except RuntimeError:
            raise _bad(f"out strides {out.stride()}: its rows have no common stride") from None
        ys = y.stride(0) if rows > 1 else n
        if ys < n:
            raise _bad(f"out strides {out.stride()}: its rows overlap")
    if save_preact:
        z = x.new_empty((*lead, wide))
        pz = z.data_ptr()
    global _c_linear
    if _c_linear is None:
        _c_linear = lib().senmoe_linear
    status = _c_linear(
        _pack_linear(code, act, groups, path, rows, k, n, x.data_ptr(), xs, weight.data_ptr(), ws, gs,
                     0 if offsets is None else offsets.data_ptr(), pb, pr, rs, y.data_ptr(), ys, pz, wide),
        _current_stream(device))
    if status:
        _check(status)
    return (out, z) if save_preact else out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, activation: str = "none", save_preact: bool = False, stream=None,
           out: torch.Tensor | None = None, path: int = LINEAR_AUTO):
    """act(x [..., in] @ weight [wide, in].T + bias [wide]) + residual [..., out] -> [..., out].

    ``save_preact`` also returns what the activation was applied to,
    [..., wide], for ``linear_backward``.
    """
    if weight.dim() != 2:
        raise _bad(f"weight must be [out, in], got {tuple(weight.shape)}")
    return _forward(x, weight, None, bias, residual, activation, save_preact, stream, out, path)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: torch.Tensor | None = None,
                   activation: str = "none", save_preact: bool = False, stream=None, out: torch.Tensor | None = None,
                   path: int = LINEAR_AUTO):
    """linear with weight [E, wide, in] and bias [E, wide] of each row's
    expert; x [S, in] in expert order, offsets int32 [E + 1].  Rows outside
    [offsets[0], offsets[E]) come out as zero."""
    if x.dim() != 2:
        raise _bad(f"x must be [rows, in], got {tuple(x.shape)}")
    _check_groups(offsets, weight, x)
    return _forward(x, weight, offsets, bias, None, activation, save_preact, stream, out, path)


def _backward(dy, x, weight, offsets, preact, activation, bias, need_dx, need_dweight, stream, path):
    if stream is not None:
        with torch.cuda.stream(stream):
            return _backward(dy, x, weight, offsets, preact, activation, bias, need_dx, need_dweight, None, path)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise _no_activation(activation)
    code, device = _operands(x, dy, weight)
    wshape, xshape = weight.shape, x.shape
    wide, k = wshape[-2], wshape[-1]
    if wide < 1 or k < 1:
        raise _bad(f"weight {tuple(wshape)}: in_features={k} out_features={wide}")
    n = wide
    if act >= _GATED:
        if wide % 2:
            raise _bad(f"{activation}: weight has {wide} rows, gate and up need an even number")
        n = wide // 2
    if not xshape or xshape[-1] != k or dy.shape != (*xshape[:-1], n):
        raise _bad(f"dy {tuple(dy.shape)} and x {tuple(xshape)} against weight {tuple(wshape)}")
    pz = zs = pws = need = 0
    if act:
        if preact is None or preact.shape != (*xshape[:-1], wide):
            raise _bad(f"{activation}: preact {None if preact is None else tuple(preact.shape)}, "
                       f"{(*xshape[:-1], wide)} wanted")
        _same(preact, x, x.dtype, device)
        preact, zs = _rows(preact, wide)
        pz = preact.data_ptr()
    groups = 1
    if offsets is not None:
        groups, offsets = wshape[0], offsets.contiguous()
    dy, dys = _rows(dy, n)
    x, xs = _rows(x, k)
    weight, ws, gs = _matrices(weight, wide, k)
    dx = x.new_empty(xshape) if need_dx else None
    dw = x.new_empty(wshape) if need_dweight else None
    db = x.new_empty(wshape[:-1]) if bias else None
    args = (code, act, groups, path, x.numel() // k, k, n, dy.data_ptr(), dys, x.data_ptr(), xs, weight.data_ptr(), ws,
            gs, 0 if offsets is None else offsets.data_ptr(), pz, zs, dx.data_ptr() if need_dx else 0, k,
            dw.data_ptr() if need_dweight else 0, k, wide * k, db.data_ptr() if bias else 0)
    L = lib()
    if act or bias:
        need = L.senmoe_linear_backward_workspace(_pack_grad(*args, 0, 0))
        if need < 0:
            _check(-need)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
            pws = workspace.data_ptr()
    status = L.senmoe_linear_backward(_pack_grad(*args, pws, need), _current_stream(device))
    if status:
        _check(status)
    return dx, dw, db


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, preact: torch.Tensor | None = None,
                    activation: str = "none", bias: bool = False, need_dx: bool = True, need_dweight: bool = True,
                    stream=None, path: int = LINEAR_AUTO):
    """(dx, dweight, dbias) of ``linear`` from dy [..., out]; dbias None
    without ``bias``, dx / dweight None where not needed.  ``preact`` is what
    ``save_preact`` returned (not used for activation ``none``)."""
    if weight.dim() != 2:
        raise _bad(f"weight must be [out, in], got {tuple(weight.shape)}")
    return _backward(dy, x, weight, None, preact, activation, bias, need_dx, need_dweight, stream, path)


def grouped_linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                            preact: torch.Tensor | None = None, activation: str = "none", bias: bool = False,
                            need_dx: bool = True, need_dweight: bool = True, stream=None, path: int = LINEAR_AUTO):
    """(dx [S, in], dweight [E, wide, in], dbias [E, wide]) of
    ``grouped_linear`` from dy [S, out].  Experts without rows get zeros."""
    if x.dim() != 2:
        raise _bad(f"x must be [rows, in], got {tuple(x.shape)}")
    _check_groups(offsets, weight, x)
    return _backward(dy, x, weight, offsets, preact, activation, bias, need_dx, need_dweight, stream, path)


def linear_check(stream=None) -> None:
    """Synchronises and raises if a bounded wait of the linear kernels ran out on this device."""
    s = torch.cuda.current_stream() if stream is None else stream
    _check(lib().senmoe_linear_check(s.cuda_stream))
