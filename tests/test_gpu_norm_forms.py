"""Forms of the norm that take particular sizes, strides or arguments to reach,
on the GPU against float64 with elementwise bounds (rows8_ref.py)."""
import pytest
from test_gpu_norm import EPS, _make

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


@pytest.mark.parametrize("n", [320, 333])
def test_backward_of_strided_rows_keeps_their_shape(senmoe, torch, n):
    """Rows of three dimensions that are no plain buffer: a slice of wider ones, transposed, expanded."""
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, 24, n, "bfloat16")
    rx, bx, rw, bw = R.norm_backward(s["dy"], s["x"], s["w"], EPS, s["dh"])
    cube = {k: s[k].view(4, 6, n) for k in ("dy", "x", "dh")}

    def sliced(t):
        wide = torch.zeros(4, 6, n + 9, dtype=t.dtype, device="cuda")
        wide[..., 1:n + 1] = t
        return wide[..., 1:n + 1]
    for form in (sliced, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        v = {k: form(t) for k, t in cube.items()}
        assert not v["x"].is_contiguous()
        dx, dw = senmoe.rms_norm_backward(v["dy"], v["x"], s["w"], EPS, dh=v["dh"])
        assert dx.shape == (4, 6, n) and dw.shape == (n,)
        L.assert_within(dx.reshape(24, n), rx, R.rounded(rx, bx, dx.dtype), "dx")
        L.assert_within(dw, rw, R.rounded(rw, bw, dw.dtype), "dweight")
    row = s["x"][:1].expand(24, n)  # one row, 24 times
    gx, _ = senmoe.rms_norm_backward(s["dy"], row, s["w"], EPS)
    assert gx.shape == (24, n) and torch.equal(gx, senmoe.rms_norm_backward(s["dy"], row.contiguous(), s["w"], EPS)[0])


@pytest.mark.parametrize("rows,n,stride", [(9, 2048, 2048), (9, 2048, 2051), (40, 333, 333), (40, 96, 101), (2, 17000, 17000)])
def test_h_without_a_residual_is_x(senmoe, torch, rows, n, stride):
    """The C entry's h is what was normed: beside another output x itself where there is no residual."""
    from senmoe import norm
    s = _make(torch, rows, n, "float16")
    want = senmoe.rms_norm(s["x"], s["w"], EPS)
    h, y = torch.zeros(rows, stride, dtype=torch.float16, device="cuda"), torch.zeros_like(s["x"])
    call = lambda py: senmoe.lib().senmoe_rms_norm(  # noqa: E731
        norm._pack_norm(1, 0, 0, EPS, rows, n, s["x"].data_ptr(), n, 0, 0, s["w"].data_ptr(), h.data_ptr(), stride, py, n,
                        0, 0, 0, 0), torch.cuda.current_stream().cuda_stream)
    assert call(0) == 1 and not bool(h.any())  # (a copy alone is refused)
    assert call(y.data_ptr()) == 0
    assert torch.equal(h[:, :n], s["x"]) and not bool(h[:, n:].any())
    if stride == n:  # (else the rows are on another grid: another kernel's sums)
        assert torch.equal(y, want.y)


# rows past which a warp's next row is on its way, with ragged last rounds: 1 to 16 warps a row, 1 to 4 pieces a lane
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,n", [(40003, 64), (20001, 256), (20003, 512), (20011, 768), (20001, 1024), (10007, 1088),
                                    (10001, 2048), (9001, 2816), (5003, 4096), (3001, 8192), (2001, 12288), (1501, 16384)])
def test_forward_of_many_rows(senmoe, torch, rows, n, residual, dtype):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, rows, n, dtype)
    r = s["r"] if residual else None
    got = senmoe.rms_norm(s["x"], s["w"], EPS, residual=r, eight_bit=True)
    y, d, h = R.norm(s["x"], s["w"], EPS, r)
    assert torch.equal(got.h, h)
    L.assert_within(got.y, y, R.rounded(y, d, h.dtype), "y")
    R.assert_rows8(got.y8, y, d, "y8")


def _off_grid(torch, t, pad=1):
    """t's values in rows that start on no 16-byte grid."""
    wide = torch.zeros(t.shape[0], t.shape[1] + 2 * pad + 1, dtype=t.dtype, device="cuda")
    wide[:, pad:pad + t.shape[1]] = t
    return wide[:, pad:pad + t.shape[1]]


# a warp a row (up to 512 columns) and a block a row, also with more rows than run at once
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,n", [(70, 320), (40001, 96), (38003, 223), (64, 544), (3001, 820), (2003, 1056), (1301, 16416)])
def test_forward_on_no_grid(senmoe, torch, rows, n, dtype):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, rows, n, dtype)
    eight = n % 32 == 0
    y, d, h = R.norm(s["x"], s["w"], EPS, s["r"])
    got = senmoe.rms_norm(_off_grid(torch, s["x"]), s["w"], EPS, residual=_off_grid(torch, s["r"], 3), eight_bit=eight)
    assert torch.equal(got.h, h)
    L.assert_within(got.y, y, R.rounded(y, d, h.dtype), "y")
    if eight:
        R.assert_rows8(got.y8, y, d, "y8")


# 1, 4 and 16 warps a row, each with one and with several rows a warp, and a block a row
@pytest.mark.parametrize("dtype,fp32", [("bfloat16", False), ("bfloat16", True), ("float16", False)])
@pytest.mark.parametrize("dh", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 513), (9001, 333), (5, 820), (3001, 820), (4001, 1467), (2500, 2047), (3, 2049),
                                    (1000, 2051), (700, 4099), (900, 8191), (601, 8193)])
def test_backward_of_odd_widths(senmoe, torch, rows, n, dh, dtype, fp32):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, rows, n, dtype, seed=8, fp32=fp32)
    extra = s["dh"] if dh else None
    dx, dw = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS, dh=extra)
    rx, bx, rw, bw = R.norm_backward(s["dy"], s["x"], s["w"], EPS, extra)
    L.assert_within(dx, rx, R.rounded(rx, bx, dx.dtype), "dx")
    L.assert_within(dw, rw, bw if fp32 else R.rounded(rw, bw, dw.dtype), "dweight")
    again = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS, dh=extra)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("rows,n", [(9001, 1024), (30001, 256), (5003, 2816), (4001, 8192), (1001, 16384)])
def test_backward_of_many_rows(senmoe, torch, rows, n):
    import linear_ref as L
    import rows8_ref as R
    s = _make(torch, rows, n, "bfloat16", seed=9)
    dx, dw = senmoe.rms_norm_backward(s["dy"], s["x"], s["w"], EPS, dh=s["dh"])
    rx, bx, rw, bw = R.norm_backward(s["dy"], s["x"], s["w"], EPS, s["dh"])
    L.assert_within(dx, rx, R.rounded(rx, bx, dx.dtype), "dx")
    L.assert_within(dw, rw, R.rounded(rw, bw, dw.dtype), "dweight")
