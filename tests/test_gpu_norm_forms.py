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
    """The C entry's h is what was normed: x itself where there is no residual, also as the call's only output."""
    from senmoe import norm
    s = _make(torch, rows, n, "float16")
    want = senmoe.rms_norm(s["x"], s["w"], EPS)
    for y in (torch.zeros_like(s["x"]), None):
        h = torch.zeros(rows, stride, dtype=torch.float16, device="cuda")
        assert senmoe.lib().senmoe_rms_norm(
            norm._pack_norm(1, 0, 0, EPS, rows, n, s["x"].data_ptr(), n, 0, 0, s["w"].data_ptr(), h.data_ptr(), stride,
                            0 if y is None else y.data_ptr(), n, 0, 0, 0, 0), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(h[:, :n], s["x"]) and not bool(h[:, n:].any())
        if y is not None and stride == n:  # (else the rows are on another grid: another kernel's sums)
            assert torch.equal(y, want.y)
