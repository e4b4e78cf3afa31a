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
