"""Rows in 8 bits and the products over them on the GPU, dense and grouped,
against float64 with elementwise bounds (rows8_ref.py)."""
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16"]
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu"]


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


@pytest.fixture(params=["small", "one", "pair", "split", "auto"])
def path(request, senmoe):
    return {"small": senmoe.LINEAR_SMALL, "one": senmoe.LINEAR_TCGEN05_ONE, "pair": senmoe.LINEAR_TCGEN05_PAIR,
            "split": senmoe.LINEAR_TCGEN05_SPLIT, "auto": senmoe.LINEAR_AUTO}[request.param]


def _same8(torch, a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def _make(senmoe, torch, rows, k, wide, dtype="bfloat16", seed=0, experts=None, std=0.7, out=None):
    import rows8_ref as R
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + k * 3 + wide)
    dt = getattr(torch, dtype)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale
    lead = () if experts is None else (experts,)
    # scales that differ from block to block and row to row
    spread = torch.exp2(torch.randint(-3, 4, (rows, k // 32), generator=g, device="cuda")).repeat_interleave(32, -1)
    s = {"x": R.rows8(senmoe, normal(rows, k) * spread),
         "w": R.rows8(senmoe, normal(*lead, wide, k, scale=std / k ** 0.5) *
                      torch.exp2(torch.randint(-2, 3, (*lead, wide, k // 32), generator=g, device="cuda")
                                 ).repeat_interleave(32, -1)),
         "b": normal(*lead, wide, scale=0.3).to(dt), "r": normal(rows, out or wide).to(dt)}
    return s


def _offsets(torch, counts, first=0):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def _wide(activation, out):
    return out * (2 if activation in ("swiglu", "geglu") else 1)


def _call(senmoe, torch, fn, *args, **kw):
    """The call, or None where the form asked for does not take this many tiles."""
    try:
        return fn(*args, **kw)
    except senmoe.SenMoeError as e:
        assert kw["path"] == senmoe.LINEAR_TCGEN05_SPLIT and e.status == 5, e
        return None


# ------------------------------------------------------------ quantize8
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 32), (1, 2048), (3, 96), (37, 704), (65, 2816), (1000, 1056), (2, 4128)])
def test_quantize(senmoe, torch, rows, n, dtype):
    import rows8_ref as R
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x = (torch.randn(rows, n, generator=g, device="cuda") *
         torch.exp2(torch.randint(-12, 13, (rows, n), generator=g, device="cuda"))).to(getattr(torch, dtype))
    got = senmoe.quantize8(x)
    want = R.rows8(senmoe, x)
    assert _same8(torch, got, want)  # every step of it is exact but the one rounding
    R.assert_rows8(got, x.double(), torch.zeros(x.shape, dtype=torch.float64, device="cuda"), "x")
    assert torch.equal(got.dequantize().double(), R.values(got))
    assert torch.equal(got.take(torch.tensor([rows - 1], device="cuda")).codes.view(torch.uint8),
                       got.codes[-1:].view(torch.uint8))


def test_quantize_borders(senmoe, torch):
    """Largest values at and beside 448 2^e, ties, subnormals, zeros, infinities, NaN, the ends of the scales' range."""
    import rows8_ref as R
    x = torch.zeros(12, 32, dtype=torch.bfloat16, device="cuda")
    x[0, 3] = 448.0
    x[1, 3] = 450.0
    x[2, 3], x[2, 4] = 448.0, 2.0 ** -10  # a tie between zero and the smallest subnormal: to even
    x[3, :] = torch.arange(32, device="cuda") * 0.5 + 240.0
    x[4, 0], x[4, 1] = -448.0, 3 * 2.0 ** -10
    x[5, 0] = 2.0 ** -126
    x[6, 0] = 1.5 * 2.0 ** 127
    x[7, 0] = 2.0 ** -133
    got = senmoe.quantize8(x)
    assert _same8(torch, senmoe.Rows8(*(t[:8] for t in got)), R.rows8(senmoe, x[:8]))
    assert torch.equal(got.dequantize()[8:], torch.zeros(4, 32, device="cuda"))
    x[9, 5] = float("inf")
    x[10, 5] = float("-inf")
    x[11, 5] = float("nan")
    v = senmoe.quantize8(x).dequantize()
    assert bool(v[9:].isnan().all()) and torch.equal(v[:9], got.dequantize()[:9])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("rows,n", [(1, 32), (19, 320), (130, 1056)])
def test_dz_in_8_bits(senmoe, torch, activation, rows, n, dtype):
    import rows8_ref as R
    from senmoe import products8
    from senmoe.products import ACTIVATIONS
    g = torch.Generator(device="cuda").manual_seed(n)
    dt = getattr(torch, dtype)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dt)
    z = (1.5 * torch.randn(rows, _wide(activation, n), generator=g, device="cuda")).to(dt)
    ref, d = R.dz(dy, z, activation)
    got = products8._quantize(dy, z, ACTIVATIONS[activation], 0)
    R.assert_rows8(got, ref, d, "dz")
    # a base off the grid: one element a lane, the same values
    pad = torch.empty(rows, z.shape[1] + 1, dtype=dt, device="cuda")
    pad[:, 1:] = z
    assert _same8(torch, products8._quantize(dy, pad[:, 1:], ACTIVATIONS[activation], 0), got)


# -------------------------------------------------------------- products
# rows, in, out: sizes at which tiles, stages, scale words and single rows end
DENSE = [(1, 32, 128), (1, 2048, 32), (2, 64, 16), (7, 96, 24), (17, 128, 129), (63, 160, 64), (64, 704, 127),
         (65, 256, 200), (129, 512, 264), (225, 544, 136), (257, 1024, 1), (300, 2816, 96), (513, 768, 256)]


@pytest.mark.parametrize("rows,k,out", DENSE)
def test_linear8_sizes(senmoe, torch, path, rows, k, out):
    import linear_ref as L
    import rows8_ref as R
    s = _make(senmoe, torch, rows, k, out)
    y = _call(senmoe, torch, senmoe.linear8, s["x"], s["w"], bias=s["b"], residual=s["r"], path=path)
    if y is None:
        return
    ref, d, _, _ = R.product(R.values(s["x"]), R.values(s["w"]), None, s["b"], s["r"])
    L.assert_within(y, ref, R.rounded(ref, d, y.dtype), "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("rows,k,out", [(1, 256, 160), (70, 192, 96), (230, 320, 288)])
def test_linear8_activations(senmoe, torch, path, activation, rows, k, out, dtype):
    import linear_ref as L
    import rows8_ref as R
    wide = _wide(activation, out)
    s = _make(senmoe, torch, rows, k, wide, dtype, std=1.5, out=out)
    dt = getattr(torch, dtype)
    kw = {"bias": s["b"], "activation": activation, "save_preact": True, "dtype": dt, "path": path}
    got = _call(senmoe, torch, senmoe.linear8, s["x"], s["w"], residual=s["r"], **kw)
    if got is None:
        return
    x, w = R.values(s["x"]), R.values(s["w"])
    ref, d, zr, zd = R.product(x, w, None, s["b"], s["r"], activation)
    L.assert_within(got[1], zr, R.rounded(zr, zd, dt), "preact")
    L.assert_within(got[0], ref, R.rounded(ref, d, dt), "y")
    y8, z = senmoe.linear8(s["x"], s["w"], eight_bit=True, **kw)
    ref, d, _, _ = R.product(x, w, None, s["b"], None, activation)
    L.assert_within(z, zr, R.rounded(zr, zd, dt), "preact beside y8")  # (the few-row kernel adds in another order)
    R.assert_rows8(y8, ref, d, "y8")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("activation", ["none", "swiglu"])
@pytest.mark.parametrize("counts,first", [([5, 0, 40, 1, 0, 130, 64, 3], 0), ([0, 0, 0, 0], 3), ([1], 0), ([300, 7], 5),
                                          ([16] * 40, 0), ([225, 224, 223, 33], 1)])
def test_grouped_linear8(senmoe, torch, path, counts, first, activation, eight):
    """Ragged groups, empty ones, rows before the first group and behind the last (zeros)."""
    import linear_ref as L
    import rows8_ref as R
    k, out = 288, 96
    rows = first + sum(counts) + 6
    wide = _wide(activation, out)
    s = _make(senmoe, torch, rows, k, wide, experts=len(counts))
    off = _offsets(torch, counts, first)
    got = _call(senmoe, torch, senmoe.grouped_linear8, s["x"], s["w"], off, bias=s["b"], activation=activation,
                save_preact=True, eight_bit=eight, path=path)
    if got is None:
        return
    y, z = got
    ref, d, zr, zd = R.product(R.values(s["x"]), R.values(s["w"]), off, s["b"], None, activation)
    L.assert_within(z, zr, R.rounded(zr, zd, z.dtype), "preact")
    if eight:
        R.assert_rows8(y, ref, d, "y8")
        y = y.codes.view(torch.uint8)
    else:
        L.assert_within(y, ref, R.rounded(ref, d, y.dtype), "y")
    for part in (slice(0, first), slice(rows - 6, rows)):
        assert not bool(y[part].any()) and not bool(z[part].any())


def test_linear8_one_by_one(senmoe, torch, path):
    """Each element of x and W alone, with its own scale: no row, column, block or scale is taken for another."""
    import rows8_ref as R
    rows, k, out = 40, 256, 160
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.zeros(rows, k, dtype=torch.float64, device="cuda")
    col = torch.randint(0, k, (rows,), generator=g, device="cuda")
    x[torch.arange(rows, device="cuda"), col] = torch.exp2(torch.randint(-20, 20, (rows,), generator=g, device="cuda").double())
    w = torch.randint(-7, 8, (out, k), generator=g, device="cuda").double()
    w *= torch.exp2(torch.randint(-20, 20, (out, k // 32), generator=g, device="cuda").double()).repeat_interleave(32, -1)
    xr, wr = R.rows8(senmoe, x), R.rows8(senmoe, w)
    assert torch.equal(R.values(wr), w)
    y = _call(senmoe, torch, senmoe.linear8, xr, wr, path=path)
    if y is None:
        return
    assert torch.equal(y.double(), x @ w.t())  # one product each: exact


def test_linear8_exact_sums(senmoe, torch, path):
    """Whole numbers whose sums need 24 bits: fp32 sums are exact, fewer bits are not."""
    rows, k, out = 33, 1024, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(0, 2, (rows, k), generator=g, device="cuda").double() * 240
    w = torch.randint(0, 2, (out, k), generator=g, device="cuda").double() * 15
    x[:, 0::32], w[:, 0::32] = 1.0, 1.0  # next to the large ones
    import rows8_ref as R
    xr, wr = R.rows8(senmoe, x), R.rows8(senmoe, w)
    assert torch.equal(R.values(xr), x) and torch.equal(R.values(wr), w)
    whole = (x @ w.t()).round()
    y = _call(senmoe, torch, senmoe.linear8, xr, wr, residual=(-whole).to(torch.bfloat16), path=path)
    if y is None:
        return
    left = whole + (-whole).to(torch.bfloat16).double()  # |left| <= 2^-8 of it: the residual takes the leading bits off
    assert torch.equal(y, left.to(torch.bfloat16))


def test_linear8_nan_scales_stay_in_their_rows(senmoe, torch, path):
    """A block that reads as NaN makes its row of y NaN and no other; infinities behind the last row reach nothing."""
    s = _make(senmoe, torch, 50, 128, 96)
    s["x"].scales.view(torch.uint8)[7, 2] = 255
    s["w"].scales.view(torch.uint8)[40, 0] = 255
    y = _call(senmoe, torch, senmoe.linear8, s["x"], s["w"], path=path)
    if y is None:
        return
    want = torch.zeros(50, 96, dtype=torch.bool, device="cuda")
    want[7] = True
    want[:, 40] = True
    assert torch.equal(y.isnan(), want)
    cut = senmoe.linear8(senmoe.Rows8(*(t[:7] for t in s["x"])), s["w"], path=path)
    assert torch.equal(cut.isnan(), want[:7])


@pytest.mark.parametrize("k", [64, 704, 2048])
def test_linear8_strides(senmoe, torch, path, k):
    """Rows of wider buffers, scales off every grid, bases off the codes' grid (copied), 3-d rows."""
    rows, out = 70, 64
    s = _make(senmoe, torch, rows, k, out)
    want = _call(senmoe, torch, senmoe.linear8, s["x"], s["w"], residual=s["r"], path=path)
    if want is None:
        return

    def inside(t, before, after):
        raw = t.view(torch.uint8)
        wide = torch.full((raw.shape[0], before + raw.shape[1] + after), 200, dtype=torch.uint8, device="cuda")
        wide[:, before:before + raw.shape[1]] = raw
        return wide[:, before:before + raw.shape[1]].view(t.dtype)
    for a, b in ((16, 32), (1, 2), (3, 1)):
        x = senmoe.Rows8(inside(s["x"].codes, a, 2 * b), inside(s["x"].scales, b, a))
        w = senmoe.Rows8(inside(s["w"].codes, 2 * b, a), inside(s["w"].scales, a, b))
        assert torch.equal(senmoe.linear8(x, w, residual=s["r"], path=path), want)
    cube = senmoe.linear8(senmoe.Rows8(*(t.view(2, 35, -1) for t in s["x"])), s["w"], residual=s["r"].view(2, 35, out), path=path)
    assert torch.equal(cube.view(rows, out), want)
    t = senmoe.Rows8(s["x"].codes.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn), s["x"].scales)
    assert torch.equal(senmoe.linear8(t, s["w"], residual=s["r"], path=path), want)


def test_grouped_linear8_slice_of_experts(senmoe, torch, path):
    """A rank's own experts: a slice of the weights and of the offsets."""
    counts = [9, 33, 0, 50, 21, 2]
    s = _make(senmoe, torch, sum(counts), 160, 64, experts=6)
    off = _offsets(torch, counts)
    whole = _call(senmoe, torch, senmoe.grouped_linear8, s["x"], s["w"], off, path=path)
    if whole is None:
        return
    part = senmoe.grouped_linear8(s["x"], senmoe.Rows8(s["w"].codes[2:5], s["w"].scales[2:5]), off[2:6], path=path)
    lo, hi = int(off[2]), int(off[5])
    assert torch.equal(part[lo:hi], whole[lo:hi])
    assert not bool(part[:lo].any()) and not bool(part[hi:].any())


def test_grouped_linear8_bad_offsets_touch_nothing_else(senmoe, torch):
    """Offsets that decrease or leave the rows are clamped: no fault, and what lies around y stays."""
    rows, k, out = 40, 64, 32
    s = _make(senmoe, torch, rows, k, out, experts=3)
    for values in ([0, 30, 10, 40], [-5, 10, 20, 400], [50, 60, 70, 80], [2 ** 31 - 1, 0, -2 ** 31, 7]):
        off = torch.tensor(values, dtype=torch.int32, device="cuda")
        for path in (senmoe.LINEAR_SMALL, senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR):
            senmoe.grouped_linear8(s["x"], s["w"], off, path=path)
            senmoe.grouped_linear8(s["x"], s["w"], off, eight_bit=True, path=path)
    senmoe.linear_check()


# ------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["none", "gelu", "swiglu", "geglu"])
@pytest.mark.parametrize("rows,n,k", [(1, 64, 100), (67, 96, 136), (260, 320, 257)])
def test_input_grad(senmoe, torch, path, activation, rows, n, k, dtype):
    import linear_ref as L
    import rows8_ref as R
    from senmoe import products8
    from senmoe.products import ACTIVATIONS
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    dt, wide = getattr(torch, dtype), _wide(activation, n)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dt)
    z = torch.randn(rows, wide, generator=g, device="cuda").to(dt)
    wt = R.rows8(senmoe, torch.randn(k, wide, generator=g, device="cuda") / wide ** 0.5)
    dx = _call(senmoe, torch, senmoe.linear8_input_grad, dy, wt, preact=z, activation=activation, path=path)
    if dx is None:
        return
    dz = products8._quantize(dy, z, ACTIVATIONS[activation], 0)  # (held to float64 by test_dz_in_8_bits)
    ref, d, _, _ = R.product(R.values(dz), R.values(wt))
    assert dx.dtype is dt
    L.assert_within(dx, ref, R.rounded(ref, d, dt), "dx")


def test_grouped_input_grad(senmoe, torch, path):
    import linear_ref as L
    import rows8_ref as R
    from senmoe import products8
    counts = [30, 0, 5, 70, 1]
    rows, n, k = 110, 96, 200
    g = torch.Generator(device="cuda").manual_seed(9)
    dy = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    z = torch.randn(rows, 2 * n, generator=g, device="cuda").bfloat16()
    wt = R.rows8(senmoe, torch.randn(5, k, 2 * n, generator=g, device="cuda") / 14)
    off = _offsets(torch, counts)
    dx = _call(senmoe, torch, senmoe.grouped_linear8_input_grad, dy, wt, off, preact=z, activation="swiglu", path=path)
    if dx is None:
        return
    ref, d, _, _ = R.product(R.values(products8._quantize(dy, z, 5, 0)), R.values(wt), off)
    L.assert_within(dx, ref, R.rounded(ref, d, dx.dtype), "dx")
    assert not bool(dx[106:].any())


# ----------------------------------------------------------------- calls
def test_linear8_no_rows(senmoe, torch, path):
    s = _make(senmoe, torch, 4, 64, 32, experts=2)
    none = senmoe.Rows8(*(t[:0] for t in s["x"]))
    y, z = senmoe.linear8(none, senmoe.Rows8(s["w"].codes[0], s["w"].scales[0]), eight_bit=True, save_preact=True, path=path)
    assert y.codes.shape == (0, 32) and y.scales.shape == (0, 1) and z.shape == (0, 32)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert senmoe.grouped_linear8(none, s["w"], off, path=path).shape == (0, 32)
    assert senmoe.quantize8(torch.empty(0, 64, dtype=torch.float16, device="cuda")).scales.shape == (0, 2)
    assert senmoe.linear8_input_grad(torch.empty(0, 64, dtype=torch.float16, device="cuda"),
                                     senmoe.Rows8(s["w"].codes[0], s["w"].scales[0]), path=path).shape == (0, 32)


def test_linear8_repeats_streams_and_graph(senmoe, torch, path):
    """The same bits again, on another stream beside a second call, and captured with the quantization before it."""
    s = _make(senmoe, torch, 96, 512, 256, out=128)
    kw = {"activation": "swiglu", "eight_bit": True, "path": path}
    want = _call(senmoe, torch, senmoe.linear8, s["x"], s["w"], **kw)
    if want is None:
        return
    assert _same8(torch, senmoe.linear8(s["x"], s["w"], **kw), want)
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
        got += [senmoe.linear8(s["x"], s["w"], stream=side, **kw) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(_same8(torch, v, want) for v in got)
    x16 = torch.zeros(96, 512, dtype=torch.bfloat16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x8 = senmoe.quantize8(x16)
        out = senmoe.linear8(x8, s["w"], **kw)
    x16.copy_(s["x"].dequantize(torch.bfloat16))
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert _same8(torch, x8, senmoe.quantize8(x16))
    assert _same8(torch, out, senmoe.linear8(x8, s["w"], **kw))
    senmoe.linear_check()


def test_linear8_large(senmoe, torch):
    """A call of many tiles on every form against one another and, in part, float64."""
    import linear_ref as L
    import rows8_ref as R
    s = _make(senmoe, torch, 4100, 1056, 2056)
    part = slice(3000, 3100)
    ref, d, _, _ = R.product(R.values(s["x"])[part], R.values(s["w"]))
    for path in (senmoe.LINEAR_AUTO, senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR, senmoe.LINEAR_SMALL):
        y = senmoe.linear8(s["x"], s["w"], path=path)
        L.assert_within(y[part], ref, R.rounded(ref, d, y.dtype), "y")
    senmoe.linear_check()


def test_refusals(senmoe, torch):
    """What does not fit together raises before a launch, with the package's errors."""
    s = _make(senmoe, torch, 8, 64, 48, experts=2)
    x, w3 = s["x"], s["w"]
    w = senmoe.Rows8(w3.codes[0], w3.scales[0])
    x16 = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    off = _offsets(torch, [4, 4])
    bad = [lambda: senmoe.linear8(x, w3), lambda: senmoe.grouped_linear8(x, w, off),
           lambda: senmoe.linear8(senmoe.Rows8(x.codes, x.scales[:, :1]), w),
           lambda: senmoe.linear8(senmoe.Rows8(x.codes[:, :32], x.scales[:, :1]), w),
           lambda: senmoe.linear8(x, senmoe.Rows8(w.codes[:47], w.scales[:47]), activation="swiglu"),
           lambda: senmoe.linear8(x, w, bias=x16[0]), lambda: senmoe.linear8(x, w, residual=x16),
           lambda: senmoe.grouped_linear8(x, w3, off[:2]), lambda: senmoe.linear8_input_grad(x16, w, activation="silu"),
           lambda: senmoe.linear8_input_grad(x16, w, preact=x16[:4], activation="silu"),
           lambda: senmoe.linear8_input_grad(x16, w3), lambda: senmoe.linear8_input_grad(x16[:, :32], w),
           lambda: senmoe.grouped_linear8_input_grad(x16, w3, off[:2]), lambda: senmoe.linear8(x, w, path=9),
           lambda: senmoe.rms_norm(x16, x16[0, :32]), lambda: senmoe.rms_norm(x16, x16[0], residual=x16[:4]),
           lambda: senmoe.rms_norm(x16, x16[0], sixteen_bit=False), lambda: senmoe.rms_norm(x16, x16[0], eps=-1.0),
           lambda: senmoe.rms_norm_backward(x16[:4], x16, x16[0])]
    for i, call in enumerate(bad):
        with pytest.raises(senmoe.SenMoeError) as e:
            call()
        assert e.value.status == 1, i
    unsupported = [lambda: senmoe.quantize8(x16[:, :40]), lambda: senmoe.linear8(x, w, eight_bit=True),
                   lambda: senmoe.rms_norm(x16[:, :40], x16[0, :40], eight_bit=True),
                   lambda: senmoe.linear8(x, w, path=senmoe.LINEAR_ANY),
                   lambda: senmoe.linear8_input_grad(x16[:, :40], w)]
    for i, call in enumerate(unsupported):
        with pytest.raises(senmoe.SenMoeError) as e:
            call()
        assert e.value.status in (1, 5), i
    wrong = [lambda: senmoe.linear8(senmoe.Rows8(x.codes.view(torch.uint8), x.scales), w),
             lambda: senmoe.linear8(senmoe.Rows8(x.codes.cpu(), x.scales.cpu()), w),
             lambda: senmoe.linear8(x, senmoe.Rows8(w.codes.cpu(), w.scales.cpu())),
             lambda: senmoe.linear8(x, w, bias=s["b"][0].half()), lambda: senmoe.linear8(x, w, dtype=torch.float32),
             lambda: senmoe.grouped_linear8(x, w3, off.long()), lambda: senmoe.grouped_linear8(x, w3, off.cpu()),
             lambda: senmoe.rms_norm(x16, x16[0].half()), lambda: senmoe.rms_norm(x16, x16[0], residual=x16.half())]
    for i, call in enumerate(wrong):
        with pytest.raises(TypeError):
            call()
    torch.cuda.synchronize()


def test_offsets_past_32_bits(senmoe, torch):
    """Rows some 2^23 elements apart, in all over 2^32 bytes: norm, quantization and product of the last rows."""
    import rows8_ref as R
    rows, n, far = 300, 256, 1 << 23
    g = torch.Generator(device="cuda").manual_seed(3)
    buf = torch.empty(rows * far, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((rows, n), (far, 1))
    x.copy_(torch.randn(rows, n, generator=g, device="cuda"))
    w = R.rows8(senmoe, torch.randn(96, n, generator=g, device="cuda"))
    near = x.contiguous()
    gain = torch.rand(n, generator=g, device="cuda").bfloat16()
    a, b = senmoe.rms_norm(x, gain, residual=x, eight_bit=True), senmoe.rms_norm(near, gain, residual=near, eight_bit=True)
    assert torch.equal(a.y, b.y) and torch.equal(a.h, b.h) and _same8(torch, a.y8, b.y8)
    assert all(torch.equal(p, q) for p, q in zip(senmoe.rms_norm_backward(x, x, gain, dh=x), senmoe.rms_norm_backward(near, near, gain, dh=near)))
    x8 = senmoe.quantize8(x)
    assert _same8(torch, x8, senmoe.quantize8(near))
    raw = buf.view(torch.uint8)
    codes = raw.as_strided((rows, n), (2 * far, 1)).view(torch.float8_e4m3fn)
    scales = raw.as_strided((rows, n // 32), (2 * far, 1), 4096).view(torch.float8_e8m0fnu)
    codes.view(torch.uint8).copy_(x8.codes.view(torch.uint8))
    scales.view(torch.uint8).copy_(x8.scales.view(torch.uint8))
    for path in (senmoe.LINEAR_SMALL, senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR):
        assert torch.equal(senmoe.linear8(senmoe.Rows8(codes, scales), w, path=path), senmoe.linear8(x8, w, path=path))


def test_beside_the_16_bit_products(senmoe, torch):
    """8-bit and 16-bit tcgen05 kernels, every form, in turn and side by side on two streams: the same bits as alone."""
    s = _make(senmoe, torch, 700, 512, 768)
    x16, w16 = s["x"].dequantize(torch.bfloat16), s["w"].dequantize(torch.bfloat16)
    forms = (senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR, senmoe.LINEAR_AUTO)
    want8 = [senmoe.linear8(s["x"], s["w"], path=p) for p in forms]
    want16 = [senmoe.linear(x16, w16, path=p) for p in forms]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for side in (a, b):
        side.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(30):
        got.append((want8[i % 3], senmoe.linear8(s["x"], s["w"], path=forms[i % 3], stream=a)))
        got.append((want16[i % 3], senmoe.linear(x16, w16, path=forms[i % 3], stream=b if i % 2 else a)))
        got.append((want8[(i + 1) % 3], senmoe.linear8(s["x"], s["w"], path=forms[(i + 1) % 3], stream=b)))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in got)
    senmoe.linear_check()
