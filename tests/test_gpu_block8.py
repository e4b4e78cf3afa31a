"""The layer half over 8-bit rows (senmoe.block8): each step of a run against
float64 on the values that the step before it gave, and the whole against the
same block in float64 without rounding."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def senmoe():
    import build as b
    b.build()
    import senmoe as s
    return s


@pytest.fixture(scope="module")
def torch():
    import torch as t
    t.cuda.set_device(0)
    return t


def _block(senmoe, torch, T, H, I, E, K, shared, seed=0, train=True):
    from senmoe.block16 import Moe16Weights
    from senmoe.block8 import Moe8
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, fan_in=1):
        return (torch.randn(*shape, generator=g, device="cuda") / fan_in ** 0.5).bfloat16()
    w = Moe16Weights(normal(E, H, fan_in=H), normal(E, 2 * I, H, fan_in=H), normal(E, H, I, fan_in=I),
                     normal(2 * shared, H, fan_in=H) if shared else None, normal(H, shared, fan_in=shared) if shared else None)
    norm = (1 + 0.2 * torch.randn(H, generator=g, device="cuda")).bfloat16()
    return Moe8(w, norm, K, train=train), normal(T, H), normal(T, H)


def _values(rows):
    return rows.codes.double().unflatten(-1, (-1, 32)).mul(rows.scales.double()[..., None]).flatten(-2)


@pytest.mark.parametrize("T,H,I,E,K,shared", [(1, 256, 96, 8, 2, 0), (37, 320, 96, 16, 4, 64), (300, 512, 256, 8, 2, 128)])
def test_block_step_by_step(senmoe, torch, T, H, I, E, K, shared):
    import linear_ref as L
    import rows8_ref as R
    block, x, r = _block(senmoe, torch, T, H, I, E, K, shared)
    out, saved = block.forward(x, residual=r, train=True)
    n, token, offsets, prob, a, z, b, zb = saved
    w8 = block.w8
    # norm
    y, d, h = R.norm(x, block.norm, block.eps, r)
    assert torch.equal(n.h, h)
    L.assert_within(n.y, y, R.rounded(y, d, n.y.dtype), "norm")
    R.assert_rows8(n.y8, y, d, "norm in 8 bits")
    # routing
    ids, probs = senmoe.router(n.y, block.w.router, K, True)
    assert torch.equal(prob.sum(), probs.flatten()[senmoe.dispatch(ids, E)[0].long()].sum())
    # experts
    xs = _values(n.y8.take(token))
    ref, d, zr, zd = R.product(xs, _values(w8["gate_up"]), offsets, None, None, "swiglu")
    L.assert_within(z, zr, R.rounded(zr, zd, z.dtype), "gate and up")
    R.assert_rows8(a, ref, d, "activated")
    down, d, _, _ = R.product(_values(a), _values(w8["down"]), offsets)
    rows = R.rounded(down, d, x.dtype)
    want, bound = h.double(), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    want = want.index_add(0, token, down * prob[:, None].double())
    bound = bound.index_add(0, token, rows * prob[:, None].double().abs()) + (K + 2) * 2.0 ** -23 * want.abs()
    bound = R.rounded(want, bound, x.dtype)
    if shared:
        ref, d, zr, zd = R.product(_values(n.y8), _values(w8["shared_gate_up"]), None, None, None, "swiglu")
        L.assert_within(zb, zr, R.rounded(zr, zd, z.dtype), "shared gate and up")
        R.assert_rows8(b, ref, d, "shared activated")
        s, d, _, _ = R.product(_values(b), _values(w8["shared_down"]))
        want = want + s
        bound = R.rounded(want, bound + d + 2.0 ** -23 * want.abs(), x.dtype)
    L.assert_within(out, want, bound, "out")
    # the same rows one by one, and without what training keeps
    assert torch.equal(block.forward(x, residual=r).double().isfinite(), torch.ones_like(x, dtype=torch.bool))


@pytest.mark.parametrize("T,H,I,E,K,shared", [(40, 256, 96, 8, 2, 64)])
def test_block_gradients(senmoe, torch, T, H, I, E, K, shared):
    """Against float64 autograd of the block without any rounding.  Rounding to 8
    bits is off by at most 2^-4 of an element, evenly spread within a step: 2^-4 /
    sqrt(3) = 0.036 of a norm at most, and 0.6 of that over a binade's values,
    0.022.  A gradient passes at most six rounded operands (dz, W^T twice; x, W
    and a within z and the activation), whose independent errors add in squares:
    0.022 sqrt(6) = 0.054 of its norm, doubled for the norms of sums that cancel."""
    block, x, r = _block(senmoe, torch, T, H, I, E, K, shared, seed=5)
    out, saved = block.forward(x, residual=r, train=True)
    dout = (0.1 * torch.randn(T, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))).bfloat16()
    dx, grads = block.backward(dout, saved)
    senmoe.linear_check()
    n, token, offsets, prob, *_ = saved
    p = {k: getattr(block.w, k).double().requires_grad_(True) for k in ("gate_up", "down", "shared_gate_up", "shared_down")}
    p["norm"] = block.norm.double().requires_grad_(True)
    h = n.h.double().requires_grad_(True)

    def swiglu(v):
        g, u = v.chunk(2, -1)
        return g * torch.sigmoid(g) * u
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + block.eps) * p["norm"]
    o = h + swiglu(y @ p["shared_gate_up"].t()) @ p["shared_down"].t()
    for e in range(E):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        rows = swiglu(y[token[lo:hi]] @ p["gate_up"][e].t()) @ p["down"][e].t()
        o = o.index_add(0, token[lo:hi], rows * prob[lo:hi, None].double())
    want = torch.autograd.grad(o, [h, *p.values()], dout.double())
    for name, got, ref in zip(["dx", *p], [dx, *(grads[k] for k in p)], want):
        off = float((got.double() - ref).norm() / ref.norm())
        assert off <= 0.11, (name, off)
    assert float((out.double() - o.detach()).norm() / (o - h).detach().norm()) <= 0.11


def test_block_capture_and_requantize(senmoe, torch):
    """A decode step captured and replayed on other rows; new weights show after requantize."""
    block, x, r = _block(senmoe, torch, 4, 256, 64, 8, 2, 64, train=False)
    buf, res = torch.zeros_like(x), torch.zeros_like(r)
    block.forward(buf, residual=res)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block.forward(buf, residual=res)
    buf.copy_(x)
    res.copy_(r)
    g.replay()
    want = block.forward(x, residual=r)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    block.w.down.zero_()
    block.w.shared_down.zero_()
    block.requantize()
    assert torch.equal(block.forward(x, residual=r), x + r)
    with pytest.raises(ValueError):
        block.backward(x, None)


def test_block_replay_after_requantize(senmoe, torch):
    """A captured step reads the weights that requantize made, not the ones it was captured with."""
    block, x, r = _block(senmoe, torch, 4, 256, 64, 8, 2, 64)
    block.forward(x, residual=r)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block.forward(x, residual=r)
    g.replay()
    before = out.clone()
    for m in (block.w.gate_up, block.w.down, block.w.shared_gate_up, block.w.shared_down):
        m.mul_(0.5)
    block.requantize()
    other = senmoe.quantize8(block.w.gate_up.flip(0))  # (what was freed is written by others)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, block.forward(x, residual=r)) and not torch.equal(out, before)
    same = senmoe.quantize8(block.w.down.transpose(-1, -2).contiguous())
    assert torch.equal(block.w8["down_t"].codes.view(torch.uint8), same.codes.view(torch.uint8)) and other.codes.numel()
    assert torch.equal(block.w8["down_t"].scales.view(torch.uint8), same.scales.view(torch.uint8))


def test_block_without_tokens(senmoe, torch):
    block, x, r = _block(senmoe, torch, 4, 256, 64, 8, 2, 64)
    out, saved = block.forward(x[:0], residual=r[:0], train=True)
    assert out.shape == (0, 256) and not saved[2].any()
    dx, grads = block.backward(out, saved)
    torch.cuda.synchronize()
    assert dx.shape == (0, 256)
    for name, grad in grads.items():
        assert not grad.any(), name


def test_block_without_a_shared_expert_or_residual(senmoe, torch):
    block, x, _ = _block(senmoe, torch, 9, 256, 64, 8, 2, 0)
    out, saved = block.forward(x, train=True)
    assert saved[0].h is x and torch.equal(out, block.forward(x))
    dx, grads = block.backward(out, saved)
    assert dx.shape == x.shape and sorted(grads) == ["down", "gate_up", "norm"]
    with pytest.raises(senmoe.SenMoeError):
        _block(senmoe, torch, 4, 256, 48, 8, 2, 0)  # 48 columns: not whole blocks of 32
