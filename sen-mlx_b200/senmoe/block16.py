"""A mixture-of-experts block over 16-bit weights, forward and backward.

The block of deepseek_v2.rs:520-553 (router, dispatch, SwiGLU experts, weighted
combine, shared expert) for checkpoints whose experts are not quantized, and
for fine-tuning them: ``router`` and ``dispatch`` as in the quantized block,
the experts' products through ``grouped_linear``, the shared expert's through
``linear`` with the combined rows as its residual.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import dispatch, grouped_linear, grouped_linear_backward, linear, linear_backward, router


@dataclass
class Moe16Weights:
    """bf16: gate rows first in gate_up; the router stays as it is in training."""
    router: torch.Tensor                        # [E, H]
    gate_up: torch.Tensor                       # [E, 2 I, H]
    down: torch.Tensor                          # [E, H, I]
    shared_gate_up: torch.Tensor | None = None  # [2 Is, H]
    shared_down: torch.Tensor | None = None     # [H, Is]


class Moe16:
    """h = x + sum_k w_k expert_k(x) + shared(x), x [T, H] bf16.

    Nothing here waits for the device, so a bounded wait that ran out in a
    product shows only in ``senmoe.linear_check``: call it where the host waits
    anyway, in training before a step's gradients are used."""

    def __init__(self, weights: Moe16Weights, top_k: int, norm_topk_prob: bool = True):
        self.w, self.top_k, self.norm = weights, top_k, norm_topk_prob

    def forward(self, x: torch.Tensor, train: bool = False):
        """h, or with ``train`` (h, what ``backward`` needs)."""
        w, K = self.w, self.top_k
        ids, prob = router(x, w.router, K, self.norm)
        perm, inverse, offsets, _ = dispatch(ids, w.router.shape[0])
        token = torch.div(perm, K, rounding_mode="floor").long()
        xs = x[token]  # the tokens' rows in expert order
        a = grouped_linear(xs, w.gate_up, offsets, activation="swiglu", save_preact=train)
        a, z = a if train else (a, None)
        d = grouped_linear(a, w.down, offsets)
        rows = d[inverse.long()].view(x.shape[0], K, -1)
        h = (x.float() + (rows.float() * prob[..., None]).sum(1)).to(x.dtype)
        b = zb = None
        if w.shared_gate_up is not None:
            b = linear(x, w.shared_gate_up, activation="swiglu", save_preact=train)
            b, zb = b if train else (b, None)
            h = linear(b, w.shared_down, residual=h)
        saved = (x, token, xs, offsets, prob.flatten()[perm.long()], a, z, b, zb)
        return (h, saved) if train else h

    def backward(self, dh: torch.Tensor, saved):
        """(dx, gradients by name) from dh [T, H]; the routing weights are held fixed."""
        w = self.w
        x, token, xs, offsets, prob, a, z, b, zb = saved
        grads = {}
        dx = dh.float()
        if b is not None:
            db, grads["shared_down"], _ = linear_backward(dh, b, w.shared_down)
            d, grads["shared_gate_up"], _ = linear_backward(db, x, w.shared_gate_up, preact=zb, activation="swiglu")
            dx = dx + d.float()
        dd = (dh[token].float() * prob[:, None]).to(dh.dtype)
        da, grads["down"], _ = grouped_linear_backward(dd, a, w.down, offsets)
        dxs, grads["gate_up"], _ = grouped_linear_backward(da, xs, w.gate_up, offsets, preact=z, activation="swiglu")
        return dx.index_add(0, token, dxs.float()).to(dh.dtype), grads
