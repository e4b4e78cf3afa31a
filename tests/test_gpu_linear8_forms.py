"""Forms of the 8-bit products that take particular sizes to reach, against
float64 with elementwise bounds (rows8_ref.py)."""
import pytest
from test_gpu_linear8 import _make, _offsets, _same8, _wide

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


@pytest.mark.parametrize("activation", ["none", "swiglu"])
@pytest.mark.parametrize("k", [256, 512, 1024, 1536, 2560])
def test_split_over_few_blocks(senmoe, torch, k, activation):
    """A K split with CTAs that hold no block of 256 k, or an odd one, where the scale rows come by TMA (K 512, 1024,
    1536, 2560) and where they do not; often, and beside other calls."""
    import linear_ref as L
    import rows8_ref as R
    out = 64
    wide = _wide(activation, out)
    s = _make(senmoe, torch, 16, k, wide, out=out)
    ref, d, _, _ = R.product(R.values(s["x"]), R.values(s["w"]), None, s["b"], s["r"], activation)
    kw = {"activation": activation, "path": senmoe.LINEAR_TCGEN05_SPLIT}
    y = senmoe.linear8(s["x"], s["w"], bias=s["b"], residual=s["r"], **kw)
    L.assert_within(y, ref, R.rounded(ref, d, y.dtype), "y")
    for _ in range(50):
        again = senmoe.linear8(s["x"], s["w"], bias=s["b"], residual=s["r"], **kw)
        beside = senmoe.linear8(s["x"], s["w"], eight_bit=True, **kw)
    assert torch.equal(again, y) and _same8(torch, beside, senmoe.linear8(s["x"], s["w"], eight_bit=True, **kw))
    g = _make(senmoe, torch, 21, k, wide, experts=3, seed=1)
    off = _offsets(torch, [9, 0, 7], 2)
    y = senmoe.grouped_linear8(g["x"], g["w"], off, bias=g["b"], **kw)
    ref, d, _, _ = R.product(R.values(g["x"]), R.values(g["w"]), off, g["b"], None, activation)
    L.assert_within(y, ref, R.rounded(ref, d, y.dtype), "y grouped")
    senmoe.linear_check()
