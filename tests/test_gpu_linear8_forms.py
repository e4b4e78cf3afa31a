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


@pytest.fixture(params=["small", "one", "pair", "split", "auto"])
def path(request, senmoe):
    return {"small": senmoe.LINEAR_SMALL, "one": senmoe.LINEAR_TCGEN05_ONE, "pair": senmoe.LINEAR_TCGEN05_PAIR,
            "split": senmoe.LINEAR_TCGEN05_SPLIT, "auto": senmoe.LINEAR_AUTO}[request.param]


@pytest.mark.parametrize("rows", [1, 9, 40])
def test_scales_over_their_whole_range(senmoe, torch, path, rows):
    """Scales from 2^-127 to 2^127 on both sides, one element of each row of x: the product of two scales leaves fp32
    in every direction, while the result is zero, or in range, or not.  One product each, so exact."""
    k, out = 256, 96
    g = torch.Generator(device="cuda").manual_seed(rows)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")
    col = whole(0, k, rows)
    x = torch.zeros(rows, k, device="cuda")
    x[torch.arange(rows, device="cuda"), col] = whole(1, 8, rows).float()
    w = whole(-7, 8, out, k).float()
    xs, ws = whole(0, 255, rows, k // 32).to(torch.uint8), whole(0, 255, out, k // 32).to(torch.uint8)
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    y = senmoe.linear8(senmoe.Rows8(x.to(e4m3), xs.view(e8m0)), senmoe.Rows8(w.to(e4m3), ws.view(e8m0)), path=path)
    wide = lambda v, s: v.double() * torch.exp2(s.double() - 127).repeat_interleave(32, -1)  # noqa: E731
    want = wide(x, xs) @ wide(w, ws).t()
    assert not bool(y.isnan().any())
    near = (want == 0) | (want.abs() >= 2.0 ** -120)  # (what rounds to subnormals, or below them, is small)
    assert torch.equal(y[near], want.to(y.dtype)[near])
    assert bool((y[~near].abs() <= 2.0 ** -119).all())
    assert bool((want.abs() > 1e39).any()) or rows == 1


def test_zero_times_large_scales(senmoe, torch, path):
    """2^110 in a column of x, 2^40 in another one of W: the product is 0."""
    import rows8_ref as R
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(32, 64, device="cuda")
    x[:, 0], w[:, 1] = 2.0 ** 110, 2.0 ** 40
    y = senmoe.linear8(R.rows8(senmoe, x), R.rows8(senmoe, w), path=path)
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "swiglu", "geglu"])
def test_slopes_fall_on_the_right_side_of_a_border(senmoe, torch, activation):
    """dz in 8 bits against its definition in float64, element for element.  With fp32 values off by 2^-22 of themselves
    on average (activations of a few units in the last place), and borders at least 2^-4 of a value apart, at most
    2 * 2^-22 / 2^-4 = 2^-17 of the elements are rounded to the other side of one."""
    import linear_ref as L
    import rows8_ref as R
    from senmoe import products8
    from senmoe.products import ACTIVATIONS
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, n = 4096, 2048 // (2 if activation in L.GATED else 1)
    dy = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    z = torch.randn(rows, _wide(activation, n), generator=g, device="cuda").bfloat16()
    got = products8._quantize(dy, z, ACTIVATIONS[activation], 0)
    codes, scales = R.quantize(L.slope_dz(dy, z, activation))
    off = int((got.codes.double() != codes).sum())
    assert off <= codes.numel() * 2.0 ** -17, off
    assert torch.equal(got.scales.double(), scales)


def test_gelu_falls_on_the_right_side_of_a_border(senmoe, torch, path):
    """gelu in 8 bits where z is exact (one product a sum): as above."""
    import linear_ref as L
    import rows8_ref as R
    rows, k, out = 60, 32, 4096
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.zeros(rows, k, device="cuda")
    x[:, 5] = torch.randint(1, 16, (rows,), generator=g, device="cuda").float()
    w = torch.randint(-15, 16, (out, k), generator=g, device="cuda").float() * 2.0 ** -6
    xr, wr = R.rows8(senmoe, x), R.rows8(senmoe, w)
    b = torch.randn(out, generator=g, device="cuda").bfloat16()  # (its sum with z: rounded once, 2^-24)
    try:
        y = senmoe.linear8(xr, wr, bias=b, activation="gelu", eight_bit=True, path=path)
    except senmoe.SenMoeError as e:
        assert path == senmoe.LINEAR_TCGEN05_SPLIT and e.status == 5
        pytest.skip("too many tiles for a K split")
    codes, scales = R.quantize(L.act("gelu", R.values(xr) @ R.values(wr).t() + b.double()))
    off = int((y.codes.double() != codes).sum())
    assert off <= max(1, codes.numel() * 2.0 ** -17) and torch.equal(y.scales.double(), scales), off


def _grouped(senmoe, torch, *args, **kw):
    try:
        return senmoe.grouped_linear8(*args, **kw)
    except senmoe.SenMoeError as e:
        assert kw["path"] == senmoe.LINEAR_TCGEN05_SPLIT and e.status == 5, e
        pytest.skip("too many tiles for a K split")


# scale rows by TMA (K 512, 2048, 3584), in words of 8 (768) and 4 bytes (1408), and byte by byte (704)
@pytest.mark.parametrize("activation,eight", [("none", False), ("swiglu", True), ("geglu", False)])
@pytest.mark.parametrize("k", [512, 704, 768, 1408, 2048, 3584])
@pytest.mark.parametrize("counts,first", [([5, 0, 33, 1, 3], 0), ([300, 0, 161, 225, 17], 3)])
def test_grouped_scale_rows(senmoe, torch, path, counts, first, k, activation, eight):
    """Grouped calls whose scales come in several units, by each way, over ragged and empty groups."""
    import linear_ref as L
    import rows8_ref as R
    rows, out = first + sum(counts) + 5, 160
    s = _make(senmoe, torch, rows, k, _wide(activation, out), experts=len(counts))
    off = _offsets(torch, counts, first)
    y, z = _grouped(senmoe, torch, s["x"], s["w"], off, bias=s["b"], activation=activation, save_preact=True, eight_bit=eight,
                    path=path)
    ref, d, zr, zd = R.product(R.values(s["x"]), R.values(s["w"]), off, s["b"], None, activation)
    L.assert_within(z, zr, R.rounded(zr, zd, z.dtype), "preact")
    if eight:
        R.assert_rows8(y, ref, d, "y8")
        y = y.codes.view(torch.uint8)
    else:
        L.assert_within(y, ref, R.rounded(ref, d, y.dtype), "y")
    for part in (slice(0, first), slice(rows - 5, rows)):
        assert not bool(y[part].any()) and not bool(z[part].any())
    senmoe.linear_check()


@pytest.mark.parametrize("activation,eight", [("none", False), ("swiglu", True)])
@pytest.mark.parametrize("k", [96, 512])
def test_more_tiles_than_a_cta_keeps(senmoe, torch, k, activation, eight):
    """1024 experts with one to three rows: more than 64 tiles for each CTA, or pair of them."""
    import linear_ref as L
    import rows8_ref as R
    out = 1408 if activation == "none" else 704
    g = torch.Generator(device="cuda").manual_seed(5)
    counts = torch.randint(1, 4, (1024,), generator=g, device="cuda").tolist()
    s = _make(senmoe, torch, sum(counts), k, _wide(activation, out), experts=1024)
    off = _offsets(torch, counts)
    ref, d, _, _ = R.product(R.values(s["x"]), R.values(s["w"]), off, s["b"], None, activation)
    for path in (senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR, senmoe.LINEAR_AUTO):
        y = senmoe.grouped_linear8(s["x"], s["w"], off, bias=s["b"], activation=activation, eight_bit=eight, path=path)
        if eight:
            R.assert_rows8(y, ref, d, "y8")
        else:
            L.assert_within(y, ref, R.rounded(ref, d, y.dtype), "y")
    senmoe.linear_check()


def test_weights_past_32_bits(senmoe, torch):
    """Experts' weights and scales some 2^31 bytes apart."""
    import rows8_ref as R
    rows, k, out, far = 60, 512, 160, (1 << 31) + 16
    s = _make(senmoe, torch, rows, k, out, experts=3)
    off = _offsets(torch, [11, 40, 9])
    raw = torch.empty(3 * far, dtype=torch.uint8, device="cuda")
    codes, scales = raw.as_strided((3, out, k), (far, k, 1)), raw.as_strided((3, out, k // 32), (far, 16, 1), out * k)
    codes.copy_(s["w"].codes.view(torch.uint8))
    scales.copy_(s["w"].scales.view(torch.uint8))
    w = senmoe.Rows8(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))
    for path in (senmoe.LINEAR_SMALL, senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR):
        want = senmoe.grouped_linear8(s["x"], s["w"], off, path=path)
        assert torch.equal(senmoe.grouped_linear8(s["x"], w, off, path=path), want)
        assert bool(R.values(s["x"]).any()) and bool(want[-1].any())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("values", [[0, 30, 10, 40], [-5, 10, 20, 400], [50, 60, 70, 80], [2 ** 31 - 1, 0, -2 ** 31, 7],
                                    [3, 9, 9, 31]])
def test_offsets_of_any_value_leave_the_buffers_around(senmoe, torch, values, eight):
    """Through the C entry, with outputs inside larger buffers: whatever the offsets hold, nothing else is written."""
    from senmoe import products8
    rows, k, out, pad = 40, 64, 32, 7
    wide = 2 * out
    s = _make(senmoe, torch, rows, k, wide, experts=3)
    off = torch.tensor(values, dtype=torch.int32, device="cuda")

    def around(cols, dtype, step):
        """[rows, cols] inside a wider and longer buffer of bytes 165, and what of it lies outside."""
        buf = torch.zeros(rows + 2 * pad, cols + step, dtype=dtype, device="cuda")
        buf.view(torch.uint8).fill_(165)
        outside = torch.ones(buf.shape, dtype=torch.bool, device="cuda")
        outside[pad:pad + rows, :cols] = False
        return buf, buf[pad:pad + rows, :cols], outside
    for path in (senmoe.LINEAR_SMALL, senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR):
        held = [around(wide, torch.bfloat16, 8)]  # preact
        held += [around(out, torch.uint8, 16), around(1, torch.uint8, 3)] if eight else [around(out, torch.bfloat16, 8)]
        z, y, *scales = (t for _, t, _ in held)
        py = (0, 0, y.data_ptr(), y.stride(0), scales[0].data_ptr(), scales[0].stride(0)) if eight else \
            (y.data_ptr(), y.stride(0), 0, 0, 0, 0)
        w = s["w"]
        products8._run_linear8(0, 5, 3, path, rows, k, out, s["x"].codes.data_ptr(), k, s["x"].scales.data_ptr(), 2,
                               w.codes.data_ptr(), k, wide * k, w.scales.data_ptr(), 2, wide * 2, off.data_ptr(), 0, 0, 0,
                               *py, z.data_ptr(), z.stride(0), device=0)
        torch.cuda.synchronize()
        for buf, _, outside in held:
            assert bool((buf[outside].view(torch.uint8) == 165).all())
    senmoe.linear_check()
