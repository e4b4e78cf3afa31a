"""RMS norm with the residual's addition and 8-bit output, and its gradients,
on the GPU against float64 with elementwise bounds (rows8_ref.py)."""
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16"]
EPS = 1e-6


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


def _make(torch, rows, n, dtype, seed=0, fp32=False, unit=False):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * rows + n)
    dt = getattr(torch, dtype)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale
    w = normal(n, scale=0.3) + (0.0 if unit else 1.0)
    return {"x": normal(rows, n, scale=2.0).to(dt), "r": normal(rows, n).to(dt), "w": w if fp32 else w.to(dt),
            "dy": normal(rows, n, scale=0.3).to(dt), "dh": normal(rows, n, scale=0.3).to(dt)}


# widths at which pieces, lanes, warps and rows held in registers end, odd ones (the kernel for any width) and the next
WIDTHS = [1, 7, 8, 32, 64, 96, 255, 256, 264, 1000, 1024, 1032, 2048, 2816, 4096, 5120, 8192, 16384, 16392, 16416, 20001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_norm_widths(senmoe, torch, rows, n, dtype):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, rows, n, dtype)
    eight = n % 32 == 0
    got = senmoe.rms_norm(s["x"], s["w"], EPS, residual=s["r"], eight_bit=eight)
    y, d, h = R.norm(s["x"], s["w"], EPS, s["r"])
    assert torch.equal(got.h, h)
    L.assert_within(got.y, y, R.rounded(y, d, h.dtype), "y")
    if eight:
        R.assert_rows8(got.y8, y, d, "y8")
        only = senmoe.rms_norm(s["x"], s["w"], EPS, residual=s["r"], sixteen_bit=False, eight_bit=True)
        assert only.y is None and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(only.y8, got.y8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("unit", [False, True])
@pytest.mark.parametrize("n", [96, 2048, 333])
def test_norm_weights(senmoe, torch, n, unit, fp32, dtype):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, 37, n, dtype, fp32=fp32, unit=unit)
    got = senmoe.rms_norm(s["x"], s["w"], 1e-3, unit_offset=unit, eight_bit=n % 32 == 0)
    y, d, h = R.norm(s["x"], s["w"], 1e-3, None, unit)
    assert got.h is s["x"]
    L.assert_within(got.y, y, R.rounded(y, d, h.dtype), "y")
    if n % 32 == 0:
        R.assert_rows8(got.y8, y, d, "y8")
    dx, dw = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], 1e-3, unit_offset=unit)
    rx, bx, rw, bw = R.norm_backward(s["dy"], s["x"], s["w"], 1e-3, None, unit)
    L.assert_within(dx, rx, R.rounded(rx, bx, dx.dtype), "dx")
    assert dw.dtype is s["w"].dtype
    L.assert_within(dw, rw, bw if fp32 else R.rounded(rw, bw, dw.dtype), "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 8, 100, 256, 1024, 1040, 2048, 2816, 8192, 16384, 16392, 17001])
@pytest.mark.parametrize("rows", [1, 5, 700])
def test_norm_backward_widths(senmoe, torch, rows, n, dtype):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, rows, n, dtype, seed=3)
    dx, dw = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS, dh=s["dh"])
    rx, bx, rw, bw = R.norm_backward(s["dy"], s["x"], s["w"], EPS, s["dh"])
    L.assert_within(dx, rx, R.rounded(rx, bx, dx.dtype), "dx")
    L.assert_within(dw, rw, R.rounded(rw, bw, dw.dtype), "dweight")
    alone, none = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS, dh=s["dh"], need_dweight=False)
    assert none is None and torch.equal(alone, dx)
    none, alone = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS, dh=s["dh"], need_dx=False)
    assert none is None and torch.equal(alone, dw)


def test_norm_backward_many_rows(senmoe, torch):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, 9001, 512, "bfloat16")
    dx, dw = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS)
    rx, bx, rw, bw = R.norm_backward(s["dy"], s["x"], s["w"], EPS)
    L.assert_within(dx, rx, R.rounded(rx, bx, dx.dtype), "dx")
    L.assert_within(dw, rw, R.rounded(rw, bw, dw.dtype), "dweight")
    again = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_norm_gradient_against_differences(senmoe, torch):
    """The gradient of sum(y dy) against central differences of the float64 definition."""
    import rows8_ref as R
    s = _make(torch, 2, 64, "float16")
    dx, dw = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS)

    def loss(x, w):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        return float((y * s["dy"].double()).sum())
    x, w, step = s["x"].double(), s["w"].double(), 1e-5
    for i, j in ((0, 0), (0, 63), (1, 17)):
        up, down = x.clone(), x.clone()
        up[i, j] += step
        down[i, j] -= step
        want = (loss(up, w) - loss(down, w)) / (2 * step)
        # the difference: step^2 times a third derivative below 100, and float64 over the step
        bound = 1e-7 + float(R.norm_backward(s["dy"], s["x"], s["w"], EPS)[1][i, j]) + 2.0 ** -11 * abs(want) + 2.0 ** -25
        assert abs(float(dx[i, j]) - want) <= bound
    up, down = w.clone(), w.clone()
    up[5] += step
    down[5] -= step
    want = (loss(x, up) - loss(x, down)) / (2 * step)
    assert abs(float(dw[5]) - want) <= 1e-7 + 2.0 ** -10 * abs(want)


@pytest.mark.parametrize("eight", [False, True])
def test_norm_strides_and_alignment(senmoe, torch, eight):
    """Rows of a wider buffer, odd strides, a base off the 16-byte grid, transposed and 3-d inputs: the same values."""
    s = _make(torch, 64, 320, "bfloat16")
    want = senmoe.rms_norm(s["x"], s["w"], EPS, residual=s["r"], eight_bit=eight)
    wide = torch.zeros(64, 1001, dtype=torch.bfloat16, device="cuda")
    for off in (0, 1, 8):
        a = wide.clone()
        a[:, off:off + 320] = s["x"]
        b = wide.clone()
        b[:, off + 3:off + 323] = s["r"]
        got = senmoe.rms_norm(a[:, off:off + 320], s["w"], EPS, residual=b[:, off + 3:off + 323], eight_bit=eight)
        assert torch.equal(got.h, want.h)
        # another order of the sum: a unit of the result
        assert bool(((got.y.double() - want.y.double()).abs() <= 2.0 ** -7 * want.y.double().abs()).all())
    t = senmoe.rms_norm(s["x"].t().contiguous().t(), s["w"], EPS, residual=s["r"], eight_bit=eight)
    assert torch.equal(t.y, want.y)
    cube = senmoe.rms_norm(s["x"].view(4, 16, 320), s["w"], EPS, residual=s["r"].view(4, 16, 320), eight_bit=eight)
    assert cube.y.shape == (4, 16, 320) and torch.equal(cube.y.view(64, 320), want.y)
    if eight:
        assert cube.y8.scales.shape == (4, 16, 10)
        for g in (t, cube):
            assert all(torch.equal(a.reshape(64, -1).view(torch.uint8), b.view(torch.uint8)) for a, b in zip(g.y8, want.y8))


def test_norm_edges(senmoe, torch):
    """No rows, rows of zeros, values whose square is far from one, infinities and NaN."""
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    got = senmoe.rms_norm(x, w, eight_bit=True)
    assert got.y.shape == (0, 64) and got.y8.scales.shape == (0, 2)
    dx, dw = senmoe.rms_norm_backward(x, x, w)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
    x = torch.zeros(5, 64, dtype=torch.bfloat16, device="cuda")
    x[1] = 2.0 ** -60
    x[2] = 2.0 ** 50
    x[3, 7] = float("inf")
    x[4, 40] = float("nan")
    got = senmoe.rms_norm(x, w, eight_bit=True)
    v = got.y8.dequantize()
    assert torch.equal(got.y[0], x[0]) and torch.equal(v[0], torch.zeros(64, device="cuda"))
    # eps decides: 2^-60 / sqrt(eps); one without it
    assert torch.allclose(got.y[1].float(), torch.full((64,), 2.0 ** -60 * 1e3, device="cuda"), rtol=2.0 ** -7)
    assert torch.equal(got.y[2], torch.ones_like(w)) and torch.equal(v[2], torch.ones(64, device="cuda"))
    # inf / inf: NaN, the others 0 in its row; the block with the NaN reads as NaN
    assert bool(got.y[3, 7].isnan()) and torch.equal(got.y[3, 8:], torch.zeros_like(got.y[3, 8:]))
    assert bool(v[3, :32].isnan().all()) and torch.equal(v[3, 32:], torch.zeros(32, device="cuda"))
    assert bool(got.y[4].isnan().all()) and bool(v[4].isnan().all())


def test_norm_in_place_of_the_residual(senmoe, torch):
    """The C entry may write h over the residual's rows, as a decode loop does."""
    from senmoe import norm
    for n in (2048, 2050):  # in registers, and the kernel for any width
        s = _make(torch, 9, n, "bfloat16")
        want = senmoe.rms_norm(s["x"], s["w"], EPS, residual=s["r"])
        r, y = s["r"].clone(), torch.empty_like(s["x"])
        assert senmoe.lib().senmoe_rms_norm(
            norm._pack_norm(0, 0, 0, EPS, 9, n, s["x"].data_ptr(), n, r.data_ptr(), n, s["w"].data_ptr(), r.data_ptr(), n,
                            y.data_ptr(), n, 0, 0, 0, 0), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(r, want.h) and torch.equal(y, want.y)


def test_norm_streams_and_graph(senmoe, torch):
    """On a stream of its own, and captured with its backward and replayed on other values."""
    s = _make(torch, 33, 2048, "bfloat16")
    want = senmoe.rms_norm(s["x"], s["w"], EPS, residual=s["r"], eight_bit=True)
    wx, ww = senmoe.rms_norm_backward(s["dy"], want.h, s["w"], EPS, dh=s["dh"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = senmoe.rms_norm(s["x"], s["w"], EPS, residual=s["r"], eight_bit=True, stream=side)
    gx, gw = senmoe.rms_norm_backward(s["dy"], got.h, s["w"], EPS, dh=s["dh"], stream=side)
    side.synchronize()
    assert torch.equal(got.y, want.y) and torch.equal(gx, wx) and torch.equal(gw, ww)
    buf = {k: torch.zeros_like(v) for k, v in s.items()}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = senmoe.rms_norm(buf["x"], buf["w"], EPS, residual=buf["r"], eight_bit=True)
        grads = senmoe.rms_norm_backward(buf["dy"], got.h, buf["w"], EPS, dh=buf["dh"])
    for k, v in s.items():
        buf[k].copy_(v)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.y, want.y) and torch.equal(got.h, want.h)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got.y8, want.y8))
    assert torch.equal(grads[0], wx) and torch.equal(grads[1], ww)
