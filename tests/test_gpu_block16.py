"""The 16-bit MoE block (router, dispatch, grouped and dense products) against
float64, its gradients against autograd, and the fine-tuning example.

Tolerances: a rounding to bf16 moves a tensor by at most 2^-8 / sqrt(3) =
2.3e-3 of its norm (uniform error within half a unit).  The forward rounds the
activation, the experts' rows, the combined rows, the shared activation and
the result: five, 1.2e-2.  A gradient adds the roundings of the kept
pre-activation, of dd, da and dz, and its own: at most ten, 2.3e-2.
"""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
ONE = 2.0 ** -8 / 3 ** 0.5

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))


def _reference(torch, block, x, dh):
    """float64 block and its gradients by autograd, over the kernels' routing."""
    import senmoe
    w = block.w
    ids, prob = senmoe.router(x, w.router, block.top_k, block.norm)
    names = ("gate_up", "down", "shared_gate_up", "shared_down")
    p = {n: getattr(w, n).double().requires_grad_(True) for n in names}
    xd = x.double().requires_grad_(True)

    def mlp(v, gu, dn):
        g, u = (v @ gu.t()).chunk(2, -1)
        return (torch.nn.functional.silu(g) * u) @ dn.t()
    h = xd + mlp(xd, p["shared_gate_up"], p["shared_down"])
    for e in range(w.router.shape[0]):
        t, k = torch.where(ids == e)
        if t.numel():
            h = h.index_add(0, t, mlp(xd[t], p["gate_up"][e], p["down"][e]) * prob[t, k].double()[:, None])
    grads = torch.autograd.grad(h, [xd] + [p[n] for n in names], dh.double())
    return h.detach(), grads[0], dict(zip(names, grads[1:]))


def _off(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k,shared", [(1, 256, 96, 16, 4, 64), (37, 256, 96, 16, 4, 64),
                                                                     (500, 512, 200, 12, 3, 136)])
def test_block16_against_float64(tokens, hidden, inter, experts, top_k, shared):
    import moe_finetune
    import torch
    torch.cuda.set_device(0)
    block = moe_finetune.make_block(hidden, inter, experts, top_k, shared, seed=tokens)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16)
    dh = torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16)
    h, saved = block.forward(x, train=True)
    dx, grads = block.backward(dh, saved)
    rh, rx, rg = _reference(torch, block, x, dh)
    assert _off(h, rh) <= 5 * ONE
    assert torch.equal(block.forward(x), h)
    assert _off(dx, rx) <= 10 * ONE
    for n, r in rg.items():
        assert _off(grads[n], r) <= 10 * ONE, n


def test_finetuning_lowers_the_loss():
    import moe_finetune
    import torch
    torch.cuda.set_device(0)
    sizes = (256, 96, 16, 4, 64)
    block, teacher = moe_finetune.make_block(*sizes, seed=0), moe_finetune.make_block(*sizes, seed=1)
    teacher.w.router = block.w.router
    x = torch.randn(300, 256, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    losses = moe_finetune.train(block, teacher, x, steps=12, lr=0.02)
    assert losses[-1] < 0.8 * losses[0], losses
    assert all(b <= a * 1.05 for a, b in zip(losses, losses[1:])), losses
