"""The linear products and their gradients in float64, with bounds on how far
a kernel that sums in fp32 and rounds once to 16 bits may be from them.

Bounds, elementwise, for a sum of n products p_i held in fp32:
  * accumulation, in any order, of exact products: (n + 8) * 2^-23 * sum |p_i|
    (2^-24 a step when rounding, twice that where an adder truncates);
  * the activation's intrinsics: 2^-17 of its value (a few fp32 units, growing
    with the exponent's argument, which stays below 100 here);
  * each rounding to 16 bits: half a unit, 2^-8 (bf16) or 2^-11 (fp16) of the
    value, and half of fp16's smallest subnormal.
"""
import math

import torch

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # torch.finfo(dtype).eps / 2
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
GATED = {"swiglu": "silu", "geglu": "gelu_tanh"}
MAX_SLOPE = 1.13  # of every activation here (gelu's is 1.129)
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu"]


def act(name, z):
    if name in GATED:
        g, u = z.chunk(2, -1)
        return act(GATED[name], g) * u
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def groups(offsets, rows):
    return [(0, 0, rows)] if offsets is None else [(e, int(offsets[e]), int(offsets[e + 1]))
                                                   for e in range(len(offsets) - 1)]


def _three(w):
    return w if w.dim() == 3 else w[None]


def forward(x, w, offsets=None, bias=None, residual=None, activation="none"):
    """(y, its bound, z, its bound) in float64."""
    dt, k = x.dtype, x.shape[1]
    w3 = _three(w)
    z = torch.zeros(x.shape[0], w3.shape[1], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(z)
    for e, a, b in groups(offsets, x.shape[0]):
        xe, we = x[a:b].double(), w3[e].double()
        z[a:b], size[a:b] = xe @ we.t(), xe.abs() @ we.abs().t()
        if bias is not None:
            be = _three(bias[..., None])[e, :, 0].double() if bias.dim() == 2 else bias.double()
            z[a:b] += be
            size[a:b] += be.abs()
    u, tiny = HALF_UNIT[dt], TINY[dt]
    dz = (k + 8) * 2.0 ** -23 * size
    y = act(activation, z)
    if activation in GATED:
        g, up = z.chunk(2, -1)
        dg, du = dz.chunk(2, -1)
        a = act(GATED[activation], g)
        dy = MAX_SLOPE * dg * (up.abs() + du) + a.abs() * du
    else:
        dy = dz * (1.0 if activation in ("none", "relu") else MAX_SLOPE)
    # the intrinsics' error goes with the activation's largest term, |z| (times up)
    if activation not in ("none", "relu"):
        dy = dy + 2.0 ** -17 * (y.abs() if activation != "gelu" else z.abs())
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -23 * y.abs()
    return y, dy + u * (y.abs() + dy) + tiny, z, dz + u * (z.abs() + dz) + tiny


def slope_dz(dy, preact, activation):
    """dz = dy * act'(preact), by differentiating the definition."""
    if activation == "none":
        return dy.double()
    z = preact.double().requires_grad_(True)
    return torch.autograd.grad(act(activation, z), z, dy.double())[0]


def backward(dy, x, w, offsets=None, preact=None, activation="none"):
    """(dx, bound), (dw, bound), (db, bound) in float64."""
    dt = x.dtype
    u, tiny = HALF_UNIT[dt], TINY[dt]
    w3 = _three(w)
    dz = slope_dz(dy, preact, activation)
    err = torch.zeros_like(dz)
    if activation != "none":  # dz is rounded to 16 bits; intrinsics against its terms' size
        size = dy.double().abs()
        if activation in GATED:
            g, up = preact.double().chunk(2, -1)
            size = torch.cat([size * up.abs(), size * g.abs()], -1)
        else:
            size = size * (1 + preact.double().abs())
        err = u * dz.abs() + 2.0 ** -17 * size + tiny
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros(w3.shape, dtype=torch.float64, device=x.device)
    db = torch.zeros(w3.shape[:2], dtype=torch.float64, device=x.device)
    bx, bw, bb = torch.zeros_like(dx), torch.zeros_like(dw), torch.zeros_like(db)
    n = w3.shape[1]
    for e, a, b in groups(offsets, x.shape[0]):
        d, xe, we, er = dz[a:b], x[a:b].double(), w3[e].double(), err[a:b]
        dx[a:b], dw[e], db[e] = d @ we, d.t() @ xe, d.sum(0)
        bx[a:b] = er @ we.abs() + (n + 8) * 2.0 ** -23 * ((d.abs() + er) @ we.abs())
        bw[e] = er.t() @ xe.abs() + (b - a + 8) * 2.0 ** -23 * ((d.abs() + er).t() @ xe.abs())
        bb[e] = er.sum(0) + (b - a + 8) * 2.0 ** -23 * (d.abs() + er).sum(0)

    def last(v, bound):
        return v, bound + u * (v.abs() + bound) + tiny
    if w.dim() == 2:
        dw, db, bw, bb = dw[0], db[0], bw[0], bb[0]
    return last(dx, bx), last(dw, bw), last(db, bb)


def assert_within(got, ref, bound, what=""):
    off = (got.double() - ref).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int(torch.where(bad, off / bound, torch.zeros_like(off)).flatten().argmax()) if off.numel() else 0
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound; worst at {i}: "
                             f"{got.flatten()[i].item()} for {ref.flatten()[i].item()} +- {bound.flatten()[i].item()}")
