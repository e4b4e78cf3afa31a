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
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import ERR_BAD_ARG, SenMoeError, SenMoeLinear, SenMoeLinearGrad, _check, lib

LINEAR_AUTO, LINEAR_ANY, LINEAR_TCGEN05 = 0, 1, 2
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "swiglu": 5, "geglu": 6}
_GATED = 5  # from here on: gated pairs
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _bad(message: str) -> SenMoeError:
    return SenMoeError(ERR_BAD_ARG, message)


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t [..., n] as (rows of n contiguous elements, their stride), a view where the strides allow one."""
    n = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, n)
    if t.stride(1) != 1 and n > 1 or t.stride(0) < n and t.shape[0] > 1:
        t = t.contiguous()
    return t, max(t.stride(0), n)


def _matrices(w: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """w [out, in] or [E, out, in]: (w, row stride, group stride)."""
    n, k = w.shape[-2], w.shape[-1]
    if (w.stride(-1) != 1 and k > 1 or w.stride(-2) < k and n > 1
            or w.dim() == 3 and w.shape[0] > 1 and w.stride(0) < n * w.stride(-2)):
        w = w.contiguous()
    stride = max(w.stride(-2), k)
    return w, stride, w.stride(0) if w.dim() == 3 else 0


def _on(stream):
    """Where temporaries, outputs and launches go: the given stream, or the current one."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _activation(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise _bad(f"activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def _operands(first: torch.Tensor, *others) -> int:
    """The common 16-bit dtype's code; every tensor on the current CUDA device."""
    dtype, device = first.dtype, first.device
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"tensors must be bfloat16 or float16, got {dtype}")
    if not first.is_cuda:
        raise TypeError("tensors must be CUDA tensors")
    if device.index != torch.cuda.current_device():
        raise _bad(f"tensors on {device}, current device is cuda:{torch.cuda.current_device()}")
    for t in others:
        if t is not None and (t.dtype != dtype or t.device != device):
            raise TypeError(f"tensors must share one dtype and device: {dtype} on {device}, {t.dtype} on {t.device}")
    return code


def _groups(offsets: torch.Tensor, weight: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    if weight.dim() != 3:
        raise _bad(f"weight must be [experts, out, in], got {tuple(weight.shape)}")
    if offsets.dtype != torch.int32 or offsets.device != x.device:
        raise TypeError(f"offsets must be int32 on {x.device}, got {offsets.dtype} on {offsets.device}")
    if offsets.dim() != 1 or offsets.numel() != weight.shape[0] + 1:
        raise _bad(f"offsets {tuple(offsets.shape)} for {weight.shape[0]} experts")
    return offsets.contiguous()


def _forward(x, weight, offsets, bias, residual, activation, save_preact, stream, out, path):
    act = _activation(activation)
    code = _operands(x, weight, bias, residual, out)
    wide, k = weight.shape[-2], weight.shape[-1]
    if x.dim() == 0 or x.shape[-1] != k:
        raise _bad(f"x {tuple(x.shape)} against weight {tuple(weight.shape)}")
    if act >= _GATED and wide % 2:
        raise _bad(f"{activation}: weight has {wide} rows, gate and up need an even number")
    n = wide // 2 if act >= _GATED else wide
    groups = 1 if offsets is None else weight.shape[0]
    if bias is not None:
        if bias.numel() != groups * wide or bias.shape[-1] != wide:
            raise _bad(f"bias {tuple(bias.shape)} for weight {tuple(weight.shape)}")
    shape = (*x.shape[:-1], n)
    if residual is not None and tuple(residual.shape) != shape:
        raise _bad(f"residual {tuple(residual.shape)}, the output is {shape}")
    if out is not None and (tuple(out.shape) != shape or n > 1 and out.stride(-1) != 1):
        raise _bad(f"out {tuple(out.shape)} strides {out.stride()}, the output is {shape}, its rows contiguous")
    with _on(stream):
        x2, xs = _rows(x)
        rows = x2.shape[0]
        w, ws, gs = _matrices(weight)
        bias = bias if bias is None else bias.contiguous()
        r, rs = (None, 0) if residual is None else _rows(residual)
        if out is None:
            y = torch.empty(shape, dtype=x.dtype, device=x.device)
            y2, ys = y, n
        else:
            y = out
            y2 = out if out.dim() == 2 else out.view(-1, n)
            ys = y2.stride(0) if rows > 1 else n
            if ys < n:
                raise _bad(f"out strides {out.stride()}: its rows overlap")
        z = torch.empty((*x.shape[:-1], wide), dtype=x.dtype, device=x.device) if save_preact else None
        q = SenMoeLinear(code, act, groups, path, rows, k, n, x2.data_ptr(), xs, w.data_ptr(), ws, gs,
                         None if offsets is None else offsets.data_ptr(),
                         None if bias is None else bias.data_ptr(), None if r is None else r.data_ptr(), rs,
                         y2.data_ptr(), ys, None if z is None else z.data_ptr(), wide)
        _check(lib().senmoe_linear(C.byref(q), torch.cuda.current_stream().cuda_stream))
    return (y, z) if save_preact else y


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
    offsets = _groups(offsets, weight, x)
    return _forward(x, weight, offsets, bias, None, activation, save_preact, stream, out, path)


def _backward(dy, x, weight, offsets, preact, activation, bias, need_dx, need_dweight, stream, path):
    act = _activation(activation)
    code = _operands(dy, x, weight, preact)
    wide, k = weight.shape[-2], weight.shape[-1]
    if act >= _GATED and wide % 2:
        raise _bad(f"{activation}: weight has {wide} rows, gate and up need an even number")
    n = wide // 2 if act >= _GATED else wide
    if x.dim() == 0 or x.shape[-1] != k or tuple(dy.shape) != (*x.shape[:-1], n):
        raise _bad(f"dy {tuple(dy.shape)} and x {tuple(x.shape)} against weight {tuple(weight.shape)}")
    if act and (preact is None or tuple(preact.shape) != (*x.shape[:-1], wide)):
        raise _bad(f"{activation}: preact {None if preact is None else tuple(preact.shape)}, "
                   f"{(*x.shape[:-1], wide)} wanted")
    groups = 1 if offsets is None else weight.shape[0]
    with _on(stream):
        dy2, dys = _rows(dy)
        x2, xs = _rows(x)
        w, ws, gs = _matrices(weight)
        z, zs = _rows(preact) if act else (None, 0)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_dx else None
        dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device) if need_dweight else None
        db = torch.empty(weight.shape[:-1], dtype=x.dtype, device=x.device) if bias else None
        g = SenMoeLinearGrad(code, act, groups, path, dy2.shape[0], k, n, dy2.data_ptr(), dys, x2.data_ptr(), xs,
                             w.data_ptr(), ws, gs, None if offsets is None else offsets.data_ptr(),
                             None if z is None else z.data_ptr(), zs, None if dx is None else dx.data_ptr(), k,
                             None if dw is None else dw.data_ptr(), k, wide * k,
                             None if db is None else db.data_ptr(), None, 0)
        L, p = lib(), C.byref(g)
        need = L.senmoe_linear_backward_workspace(p)
        if need < 0:
            _check(-need)
        if need:
            ws_buf = torch.empty(need, dtype=torch.uint8, device=x.device)
            g.workspace, g.workspace_bytes = ws_buf.data_ptr(), need
        _check(L.senmoe_linear_backward(p, torch.cuda.current_stream().cuda_stream))
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
    offsets = _groups(offsets, weight, x)
    return _backward(dy, x, weight, offsets, preact, activation, bias, need_dx, need_dweight, stream, path)


def linear_check(stream=None) -> None:
    """Synchronises and raises if a bounded wait of the linear kernels ran out on this device."""
    s = torch.cuda.current_stream() if stream is None else stream
    _check(lib().senmoe_linear_check(s.cuda_stream))
