"""Rows in 8 bits, the RMS norm and the products over such rows in float64,
with bounds on how far the kernels' results may be from them.

A block of 32 with the scale s: an element is rounded to three fraction bits,
off by at most 2^-4 of itself, or by half of the subnormals' step, 2^-10 s.
The scale is the smallest power of two with max <= 448 s: where the kernel's
fp32 value of the block's largest is off by d, any power of two that is right
for a value within d of it.

The fp32 values themselves: products as in linear_ref.py (accumulation (k + 8)
2^-23 sum |p_i|, activations 2^-17), and for the norm of n elements
  * sum of h^2: (n + 8) 2^-24 of it (every term is positive), its root half;
  * 1 / sqrt by the intrinsic: 2 units, 2^-22; the mean's division, the products
    with it and with g, the addition in g: 2^-22 together.
"""
import linear_ref as L
import torch

BLOCK = 32


def quantize(v):
    """float64 v [..., n] -> (elements, scales), from the definition."""
    g = v.reshape(*v.shape[:-1], -1, BLOCK)
    m, e = torch.frexp(g.abs().amax(-1))  # m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875)).clamp(min=-127)
    s = torch.ldexp(torch.ones_like(m), e)
    q = g / s[..., None]
    step = torch.ldexp(torch.ones_like(q), torch.frexp(q.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(q / step) * step).reshape(v.shape), s


def rows8(senmoe, v):
    """float v [..., n] as senmoe.Rows8."""
    q, s = quantize(v.double())
    return senmoe.Rows8(q.to(torch.float8_e4m3fn),
                        (torch.frexp(s)[1] + 126).to(torch.uint8).view(torch.float8_e8m0fnu))


def values(r):
    """What Rows8 stands for, in float64."""
    q = r.codes.double()
    return (q.reshape(*r.scales.shape, BLOCK) * r.scales.double()[..., None]).reshape(q.shape)


def assert_rows8(r, ref, d, name):
    """r is ref (float64, known to within d) in 8 bits."""
    s = r.scales.double()
    b = lambda t: t.reshape(*t.shape[:-1], -1, BLOCK)  # noqa: E731
    top, off = b(ref.abs()).amax(-1), b(d).amax(-1)
    assert bool((448.0 * s >= top - off).all()), f"{name}: a scale is too small"
    low = (448.0 * s / 2 >= top + off) & (s > 2.0 ** -127)
    assert not bool(low.any()), f"{name}: {int(low.sum())} scales are too large"
    half = torch.maximum(2.0 ** -4 * (ref.abs() + d), 2.0 ** -10 * s.repeat_interleave(BLOCK, -1))
    L.assert_within(values(r), ref, d + half, name)


def norm(x, weight, eps, residual=None, unit_offset=False):
    """(y, fp32 bound, h) in float64."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    g = weight.double() + (1.0 if unit_offset else 0.0)
    hd, n = h.double(), x.shape[-1]
    y = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps) * g
    g_off = 2.0 ** -24 * g.abs() if unit_offset else 0.0  # the sum 1 + weight
    return y, ((n + 8) * 2.0 ** -25 + 2.0 ** -21) * y.abs() + g_off, h


def norm_backward(dy, h, weight, eps, dh=None, unit_offset=False):
    """(dx, fp32 bound, dweight, fp32 bound) in float64."""
    g = weight.double() + (1.0 if unit_offset else 0.0)
    hd, y, n, rows = h.double(), dy.double(), h.shape[-1], dy.numel() // dy.shape[-1]
    r = 1.0 / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps)
    dn = y * g
    c = r * r * (dn * hd).mean(-1, keepdim=True)
    size = r * r * (dn * hd).abs().mean(-1, keepdim=True)
    rel = (n + 8) * 2.0 ** -24 + 2.0 ** -20  # sums, and r cubed
    dx = r * (dn - hd * c)
    dxb = rel * r * (dn.abs() + hd.abs() * size) + 2.0 ** -23 * dx.abs()
    if dh is not None:
        dx = dx + dh.double()
        dxb = dxb + 2.0 ** -24 * dx.abs()
    p = y * hd * r
    flat = p.reshape(-1, n)
    return dx, dxb, flat.sum(0), ((rows + 8) * 2.0 ** -24 + rel) * flat.abs().sum(0)


def rounded(ref, d, dtype):
    """The bound d of an fp32 value, with the rounding to 16 bits."""
    return d + L.HALF_UNIT[dtype] * (ref.abs() + d) + L.TINY[dtype]


def product(x, w, offsets=None, bias=None, residual=None, activation="none"):
    """x [S, k], w [.., wide, k] float64: (y, fp32 bound, z, fp32 bound)."""
    k = x.shape[1]
    w3 = w if w.dim() == 3 else w[None]
    z = torch.zeros(x.shape[0], w3.shape[1], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(z)
    for e, a, b in L.groups(offsets, x.shape[0]):
        z[a:b], size[a:b] = x[a:b] @ w3[e].t(), x[a:b].abs() @ w3[e].abs().t()
        if bias is not None:
            be = (bias if bias.dim() == 1 else bias[e]).double()
            z[a:b] += be
            size[a:b] += be.abs()
    dz = (k + 8) * 2.0 ** -23 * size
    y = L.act(activation, z)
    if activation in L.GATED:
        g, up = z.chunk(2, -1)
        dg, du = dz.chunk(2, -1)
        dy = L.MAX_SLOPE * dg * (up.abs() + du) + L.act(L.GATED[activation], g).abs() * du
    else:
        dy = dz * (1.0 if activation in ("none", "relu") else L.MAX_SLOPE)
    if activation not in ("none", "relu"):
        dy = dy + 2.0 ** -17 * (y.abs() if activation != "gelu" else z.abs())
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -23 * y.abs()
    return y, dy, z, dz


def dz(dy, preact, activation):
    """dz = dy act'(preact) in float64 and the bound of its fp32 value: the
    intrinsics' 2^-17 against its terms' size."""
    ref = L.slope_dz(dy, preact, activation)
    if activation == "none":
        return ref, torch.zeros_like(ref)
    size = dy.double().abs()
    if activation in L.GATED:
        g, up = preact.double().chunk(2, -1)
        size = torch.cat([size * up.abs(), size * g.abs()], -1)
    else:
        size = size * (1 + preact.double().abs())
    return ref, 2.0 ** -17 * size
