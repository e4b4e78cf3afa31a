"""The half of a decoder layer around the block (deepseek_v2.rs:613-620), its
products over 8-bit rows: residual add and norm, router, dispatch, SwiGLU
experts, weighted combine, shared expert, residual; forward and backward.

``h = x + residual; out = h + sum_k w_k expert_k(norm(h)) + shared(norm(h))``

The norm writes its rows in 16 bits for the router and in 8 for the experts;
the experts' first products write theirs in 8 bits for the second.  Training
keeps 16-bit weights (``Moe16Weights``), of which the 8-bit ones are made:
gradients of rows go through 8-bit products, gradients of weights through the
16-bit ones, as if rounding to 8 bits were the identity.
"""
from __future__ import annotations

import torch

from . import (Rows8, _dispatch, grouped_linear8, grouped_linear8_input_grad, grouped_linear_backward, linear8,
               linear8_input_grad, linear_backward, quantize8, rms_norm, rms_norm_backward, router)
from .block16 import Moe16Weights
from .products import _bad


class Saved(tuple):
    """What ``backward`` needs of a ``forward``; ``slots`` [T, K]: the rows, in
    expert order, of each token's experts."""
    slots: torch.Tensor


class Moe8:
    """x [T, H] bf16; norm [H] bf16 or fp32.  ``train`` also keeps the weights'
    transposes in 8 bits, for ``backward``; after a change of the 16-bit weights
    ``requantize`` makes the 8-bit ones again, in the same memory.

    Nothing here waits for the device, so ``forward`` can be captured into a CUDA
    graph (once run before): call ``senmoe.linear_check`` where the
    host waits anyway, in training before a step's gradients are used."""

    def __init__(self, weights: Moe16Weights, norm: torch.Tensor, top_k: int, eps: float = 1e-6,
                 norm_topk_prob: bool = True, train: bool = False):
        self.w, self.norm, self.top_k, self.eps, self.norm_topk = weights, norm, top_k, eps, norm_topk_prob
        self.train = train
        self.w8: dict[str, Rows8] = {}
        self.requantize()

    def requantize(self) -> None:
        for name in ("gate_up", "down", "shared_gate_up", "shared_down"):
            m = getattr(self.w, name)
            if m is not None:
                self._keep(name, quantize8(m))
                if self.train:
                    self._keep(name + "_t", quantize8(m.transpose(-1, -2).contiguous()))

    def _keep(self, name: str, new: Rows8) -> None:
        """new, where a captured ``forward`` reads it: in the place of the one before."""
        for kept, part in zip(self.w8.setdefault(name, new), new):
            if kept is not part:
                kept.view(torch.uint8).copy_(part.view(torch.uint8))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, train: bool = False):
        """out, or with ``train`` (out, what ``backward`` needs)."""
        w, w8, K = self.w, self.w8, self.top_k
        for name, t in (("x", x), ("the router's weight", w.router)):  # (the router reads bf16 whatever it is given)
            if t.dtype is not torch.bfloat16:
                raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
            if t.dim() != 2 or t.shape[1] != w.router.shape[1]:
                raise _bad(f"{name} {tuple(t.shape)}: x is [tokens, hidden], the router's weight [experts, hidden]")
        n = rms_norm(x, self.norm, self.eps, residual=residual, eight_bit=True)
        ids, prob = router(n.y, w.router, K, self.norm_topk)
        perm, inverse, offsets, _ = _dispatch(ids, w.router.shape[0])  # (the router's ids are in range)
        token = torch.div(perm, K, rounding_mode="floor").long()
        a = grouped_linear8(n.y8.take(token), w8["gate_up"], offsets, activation="swiglu", eight_bit=True,
                            save_preact=train)
        a, z = a if train else (a, None)
        d = grouped_linear8(a, w8["down"], offsets)
        slots = inverse.long().view(x.shape[0], K)
        rows = d[slots]
        out = (n.h.float() + (rows.float() * prob[..., None]).sum(1)).to(x.dtype)
        b = zb = None
        if w.shared_gate_up is not None:
            b = linear8(n.y8, w8["shared_gate_up"], activation="swiglu", eight_bit=True, save_preact=train)
            b, zb = b if train else (b, None)
            out = linear8(b, w8["shared_down"], residual=out)
        if not train:
            return out
        saved = Saved((n, token, offsets, prob.flatten()[perm.long()], a, z, b, zb))
        saved.slots = slots
        return out, saved

    def backward(self, dout: torch.Tensor, saved):
        """(dx, gradients by name) from dout [T, H]; dx is the residual's as well;
        the routing weights are held fixed."""
        if not self.train:
            raise ValueError("Moe8 was made without train=True")
        w, w8 = self.w, self.w8
        n, token, offsets, prob, a, z, b, zb = saved
        grads = {}
        dy = torch.zeros_like(dout, dtype=torch.float32)
        if b is not None:
            db = linear8_input_grad(dout, w8["shared_down_t"])
            _, grads["shared_down"], _ = linear_backward(dout, b.dequantize(dout.dtype), w.shared_down, need_dx=False)
            dy += linear8_input_grad(db, w8["shared_gate_up_t"], preact=zb, activation="swiglu").float()
            _, grads["shared_gate_up"], _ = linear_backward(db, n.y, w.shared_gate_up, preact=zb, activation="swiglu",
                                                            need_dx=False)
        dd = (dout[token].float() * prob[:, None]).to(dout.dtype)
        da = grouped_linear8_input_grad(dd, w8["down_t"], offsets)
        _, grads["down"], _ = grouped_linear_backward(dd, a.dequantize(dout.dtype), w.down, offsets, need_dx=False)
        dxs = grouped_linear8_input_grad(da, w8["gate_up_t"], offsets, preact=z, activation="swiglu")
        _, grads["gate_up"], _ = grouped_linear_backward(da, n.y[token], w.gate_up, offsets, preact=z,
                                                         activation="swiglu", need_dx=False)
        # a token's K rows in one order: the same bits every time, as atomic additions would not give
        dy = (dy + dxs[saved.slots].sum(1, dtype=torch.float32)).to(dout.dtype)
        dx, grads["norm"] = rms_norm_backward(dy, n.h, self.norm, self.eps, dh=dout)
        return dx, grads
