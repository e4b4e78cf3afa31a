"""GPU tests of the linear products' calls: streams, refusals, gradients at the
edges of their types' range and precision, against float64 (linear_ref.py)."""
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


def _normal(torch, seed, *shape, dtype="bfloat16", scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(getattr(torch, dtype))


def test_strided_offsets_on_another_stream(senmoe, torch):
    """A column of a table of offsets, written behind a long kernel on a stream
    that the launch's stream waits for; the current stream goes on allocating
    and writing right after the calls."""
    counts, k, out = [40, 0, 75, 13], 128, 96
    x, w = _normal(torch, 1, 128, k), _normal(torch, 2, 4, out, k, scale=k ** -0.5)
    dy = _normal(torch, 3, 128, out)
    off = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    want = senmoe.grouped_linear(x, w, off)
    grads = senmoe.grouped_linear_backward(dy, x, w, off, bias=True)
    table = torch.full((5, 3), 128, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        table.fill_(128)
        torch.cuda._sleep(20_000_000)
        table[:, 1] = off
        side.wait_stream(torch.cuda.current_stream())
        y = senmoe.grouped_linear(x, w, table[:, 1], stream=side)
        got = senmoe.grouped_linear_backward(dy, x, w, table[:, 1], bias=True, stream=side)
        junk = [torch.full((5,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]
        side.synchronize()
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(got, grads))
        torch.cuda.synchronize()
        del junk


@pytest.mark.parametrize("form", ["TCGEN05", "TCGEN05_ONE", "TCGEN05_PAIR", "TCGEN05_SPLIT"])
def test_gradients_of_no_rows_in_every_form(senmoe, torch, form):
    x, w, dy = _normal(torch, 1, 0, 64), _normal(torch, 2, 48, 64), _normal(torch, 3, 0, 48)
    dx, dw, db = senmoe.linear_backward(dy, x, w, bias=True, path=getattr(senmoe, "LINEAR_" + form))
    assert dx.shape == (0, 64) and dw.shape == w.shape and (dw == 0).all() and (db == 0).all()


def test_a_wait_that_runs_out_is_reported_once(senmoe, torch):
    """Recorded on one stream, reported and cleared by the first check after it
    on any stream; later calls and checks are right."""
    senmoe.linear_check()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    assert senmoe.lib().senmoe_selftest_linear_wait(a.cuda_stream) == 0
    senmoe.linear_check(b)  # not there yet
    with pytest.raises(senmoe.SenMoeError, match="ran out") as e:
        senmoe.linear_check(a)
    assert e.value.status == senmoe.ERR_TIMEOUT
    senmoe.linear_check(a)
    senmoe.linear_check(b)
    x, w = _normal(torch, 1, 300, 128), _normal(torch, 2, 96, 128)
    assert torch.isfinite(senmoe.linear(x, w)).all()
    senmoe.linear_check()


def _tail(torch, dtype):
    """Values from -12 to 6 that the type holds exactly, as z = x w with one nonzero column, and x, w."""
    dt = getattr(torch, dtype)
    z = torch.linspace(-12, 6, 3001, device="cuda").to(dt)
    x = torch.zeros(z.numel(), 8, dtype=dt, device="cuda")
    x[:, 0] = z
    w = torch.zeros(8, 8, dtype=dt, device="cuda")
    w[:, 0] = 1
    return x, w, z.double()


def _cdf(torch, z):
    """Phi(z); erfc keeps the lower tail's relative precision, which special.ndtr on the GPU does not (0 from -8.4 on)."""
    return 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)


# The activations' relative error: __expf's 2 + 1.17 |a| units at a = -72 (z =
# -12) 1.0e-5, the argument's rounding |a| 2^-24 = 4e-6, the division, the
# polynomial and the product a few units: 2^-15 covers them.
@pytest.mark.parametrize("form", ["ANY", "SMALL", "TCGEN05_ONE", "TCGEN05_PAIR", "TCGEN05_SPLIT"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gelu_keeps_its_relative_precision_in_the_lower_tail(senmoe, torch, form, dtype):
    import linear_ref as R
    x, w, z = _tail(torch, dtype)
    if form == "TCGEN05_SPLIT":  # few tiles only
        x, z = x[:500].contiguous(), z[:500]
    y = senmoe.linear(x, w, activation="gelu", path=getattr(senmoe, "LINEAR_" + form))
    ref = (z * _cdf(torch, z))[:, None].expand(-1, 8)
    u, tiny = R.HALF_UNIT[x.dtype], R.TINY[x.dtype]
    R.assert_within(y, ref, (u + 2.0 ** -15) * ref.abs() + tiny, "gelu")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gelu_slope_keeps_its_relative_precision_in_the_lower_tail(senmoe, torch, dtype):
    """dx = (dy act'(z)) W with one nonzero weight: dy's products alone, rounded to 16 bits
    at most twice.  Phi(z) and z phi(z) cancel near -0.75, so each of the two counts."""
    import linear_ref as R
    x, w, z = _tail(torch, dtype)
    rows = z.numel()
    dy = torch.zeros(rows, 8, dtype=x.dtype, device="cuda")
    dy[:, 0] = 1
    pre = z.to(x.dtype)[:, None].expand(rows, 8).contiguous()
    dx = senmoe.linear_backward(dy, x, w, preact=pre, activation="gelu", need_dweight=False)[0][:, 0]
    phi = torch.exp(-0.5 * z * z) * 0.3989422804014327
    cdf = _cdf(torch, z)
    ref = cdf + z * phi
    u, tiny = R.HALF_UNIT[x.dtype], R.TINY[x.dtype]
    R.assert_within(dx, ref, 2.01 * u * ref.abs() + 2.0 ** -15 * (cdf + z.abs() * phi) + 2 * tiny, "slope")


def _dz_and_size(torch, dy, z, activation):
    """dz in float64 and the size that the intrinsics' error, 2^-17, goes with."""
    import linear_ref as R
    size = dy.double().abs()
    if activation in R.GATED:
        g, up = z.double().chunk(2, -1)
        size = torch.cat([size * up.abs(), size * g.abs()], -1)
    else:
        size = size * (1 + z.double().abs())
    return R.slope_dz(dy, z, activation), size


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("activation", ["relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu"])
@pytest.mark.parametrize("counts,out", [([3], 136), ([19], 33), ([333], 200), ([5000], 64), ([0, 2, 40, 0, 300, 1], 72),
                                        ([70, 0, 9], 35)])
def test_bias_gradient_sums_unrounded_terms(senmoe, torch, counts, out, activation, dtype):
    """dbias is the sum of dy act'(z) held in 32 bits, rounded once: its bound
    has no term for a rounding of dz to 16 bits."""
    import linear_ref as R
    rows, wide, k = sum(counts), out * (2 if activation in R.GATED else 1), 40
    x, dy, z = (_normal(torch, i, rows, n, dtype=dtype) for i, n in ((1, k), (2, out), (3, wide)))
    if len(counts) == 1:
        w, off = _normal(torch, 4, wide, k, dtype=dtype, scale=k ** -0.5), None
        db = senmoe.linear_backward(dy, x, w, preact=z, activation=activation, bias=True)[2][None]
    else:
        w = _normal(torch, 4, len(counts), wide, k, dtype=dtype, scale=k ** -0.5)
        off = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        db = senmoe.grouped_linear_backward(dy, x, w, off, preact=z, activation=activation, bias=True)[2]
    dz, size = _dz_and_size(torch, dy, z, activation)
    for e, a, b in R.groups(None if off is None else off.tolist(), rows):
        ref, err = dz[a:b].sum(0), 2.0 ** -17 * size[a:b].sum(0)
        err = err + (b - a + 8) * 2.0 ** -23 * dz[a:b].abs().sum(0)
        R.assert_within(db[e], ref, err + R.HALF_UNIT[x.dtype] * (ref.abs() + err) + R.TINY[x.dtype], f"db {e}")


def _gradients(torch, dy, x, w, off, z, activation):
    """(ref, bound) of dx, dw and db for fp16.  dz is held to 16 bits at a power
    of two of each group's choice: to half a unit of itself, and to half of
    fp16's smallest step, 2^-25, which is taken as it is where the group's
    largest |dz| is between 2^-6 and 65504 and otherwise is at most 2^-39 of it."""
    import linear_ref as R
    u, tiny = R.HALF_UNIT[x.dtype], R.TINY[x.dtype]
    dz, size = _dz_and_size(torch, dy, z, activation)
    w3 = w if w.dim() == 3 else w[None]
    E, n, k = w3.shape
    out = [torch.zeros(s, dtype=torch.float64, device="cuda") for s in (x.shape, (E, n, k), (E, n)) for _ in range(2)]
    dx, bx, dw, bw, db, bb = out
    for e, a, b in R.groups(None if off is None else off.tolist(), x.shape[0]):
        if a == b:
            continue
        d, xe, we = dz[a:b], x[a:b].double(), w3[e].double()
        m = float(d.abs()[d.isfinite()].max())
        step = max(2.0 ** -39 * m, tiny if 2.0 ** -6.01 <= m <= 65600 else 0.0)
        near = 2.0 ** -17 * size[a:b]
        er = u * d.abs() + near + step
        dx[a:b], dw[e], db[e] = d @ we, d.t() @ xe, d.sum(0)
        bx[a:b] = er @ we.abs() + (n + 8) * 2.0 ** -23 * ((d.abs() + er) @ we.abs())
        bw[e] = er.t() @ xe.abs() + (b - a + 8) * 2.0 ** -23 * ((d.abs() + er).t() @ xe.abs())
        bb[e] = near.sum(0) + (b - a + 8) * 2.0 ** -23 * (d.abs() + near).sum(0)
    if w.dim() == 2:
        dw, bw, db, bb = dw[0], bw[0], db[0], bb[0]
    return [(v, bd + u * (v.abs() + bd) + tiny) for v, bd in ((dx, bx), (dw, bw), (db, bb))]


# dy, z, weight and x scales: dz far over 65504, dz of fp16's subnormals, and
# gradients that fit fp16 in both
RANGES = {"large": (300.0, 400.0, 1e-3, 1e-2), "small": (2.0 ** -20, 1.0, 20.0, 50.0), "unit": (0.5, 1.0, 0.1, 1.0)}


@pytest.mark.parametrize("form", ["AUTO", "ANY", "TCGEN05_ONE", "TCGEN05_PAIR", "TCGEN05_SPLIT"])
@pytest.mark.parametrize("activation,size", [("swiglu", "large"), ("geglu", "large"), ("swiglu", "small"),
                                             ("silu", "small"), ("gelu", "small"), ("relu", "small")])
@pytest.mark.parametrize("rows,k,out", [(5, 72, 40), (150, 136, 72), (70, 41, 33)])
def test_fp16_gradients_whose_dz_leaves_the_range(senmoe, torch, form, activation, size, rows, k, out):
    import linear_ref as R
    if k % 8 and form.startswith("TCGEN05"):
        pytest.skip("not on TMA's grid")
    wide = out * (2 if activation in R.GATED else 1)
    sy, sz, sw, sx = RANGES[size]
    dy, z = _normal(torch, 1, rows, out, dtype="float16", scale=sy), _normal(torch, 2, rows, wide, dtype="float16", scale=sz)
    w, x = _normal(torch, 3, wide, k, dtype="float16", scale=sw), _normal(torch, 4, rows, k, dtype="float16", scale=sx)
    got = senmoe.linear_backward(dy, x, w, preact=z, activation=activation, bias=rows != 5,
                                 path=getattr(senmoe, "LINEAR_" + form))
    refs = _gradients(torch, dy, x, w, None, z, activation)
    for v, (ref, bound), what in zip(got, refs, ("dx", "dw", "db")):
        if v is not None:
            keep = ref.abs() < 60000  # (an output past fp16's range is an infinity)
            assert keep.float().mean() > 0.9 or what == "db"  # (the large dbias is past fp16's range)
            R.assert_within(v[keep], ref[keep], bound[keep], what)
    senmoe.linear_check()


@pytest.mark.parametrize("form", ["AUTO", "ANY", "TCGEN05_ONE", "TCGEN05_PAIR", "TCGEN05_SPLIT"])
def test_fp16_groups_of_different_ranges(senmoe, torch, form):
    """Each group has its own power of two; one with an infinity keeps its other rows' dx."""
    import linear_ref as R
    counts, k, out, first = [40, 0, 33, 70, 1, 20], 72, 48, 3
    sizes = ["large", "unit", "small", "unit", "small", "large"]
    rows = sum(counts) + first + 5
    x = torch.full((rows, k), float("nan"), dtype=torch.float16, device="cuda")
    dy = torch.full((rows, out), float("inf"), dtype=torch.float16, device="cuda")
    z = torch.full((rows, 2 * out), 60000.0, dtype=torch.float16, device="cuda")
    w = torch.zeros(len(counts), 2 * out, k, dtype=torch.float16, device="cuda")
    o = [first]
    for e, (n, size) in enumerate(zip(counts, sizes)):
        sy, sz, sw, sx = RANGES[size]
        a, b = o[-1], o[-1] + n
        dy[a:b], z[a:b] = _normal(torch, 10 + e, n, out, scale=sy), _normal(torch, 20 + e, n, 2 * out, scale=sz)
        w[e], x[a:b] = _normal(torch, 30 + e, 2 * out, k, scale=sw), _normal(torch, 40 + e, n, k, scale=sx)
        o.append(b)
    off = torch.tensor(o, dtype=torch.int32, device="cuda")
    path = getattr(senmoe, "LINEAR_" + form)
    inner = slice(first, o[-1])
    loc = off - first
    for broken in (False, True):
        if broken:
            dy[o[5] + 7, 3] = float("inf")
        dx, dw, db = senmoe.grouped_linear_backward(dy, x, w, off, preact=z, activation="swiglu", bias=True, path=path)
        refs = _gradients(torch, dy[inner], x[inner], w, loc, z[inner], "swiglu")
        rows_ok = [i for i in range(o[-1] - first) if not broken or i != o[5] + 7 - first]
        groups_ok = [e for e in range(6) if not broken or e != 5]
        assert (dx[:first] == 0).all() and (dx[o[-1]:] == 0).all()
        for v, (ref, bound), keep, what in ((dx[inner], refs[0], rows_ok, "dx"), (dw, refs[1], groups_ok, "dw"),
                                            (db, refs[2], groups_ok, "db")):
            v, ref, bound = v[keep], ref[keep], bound[keep]
            fits = ref.abs() < 60000
            assert fits.float().mean() > 0.8 or what == "db"  # (the large groups' dbias is past fp16's range)
            R.assert_within(v[fits], ref[fits], bound[fits], what)
    senmoe.linear_check()


def test_a_tile_that_takes_longer_than_a_wait_may(senmoe, torch):
    """2^29 rows summed by one tile of one CTA: some 3 s, while a wait that
    nothing ends gives up after 2 s.  All but a few hundred rows are zero."""
    import linear_ref as R
    rows, k, out = 1 << 29, 16, 16
    if torch.cuda.mem_get_info()[0] < 45 << 30:
        pytest.skip("needs 34 GB")
    at = torch.cat([torch.arange(100), torch.arange(rows // 2, rows // 2 + 100), torch.arange(rows - 100, rows)]).cuda()
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(rows, out, dtype=torch.bfloat16, device="cuda")
    x[at], dy[at] = _normal(torch, 1, 300, k), _normal(torch, 2, 300, out)
    w = _normal(torch, 3, out, k)
    dw = senmoe.linear_backward(dy, x, w, need_dx=False, path=senmoe.LINEAR_TCGEN05_ONE)[1]
    senmoe.linear_check()
    (_, _), (ref, bound), (_, _) = R.backward(dy[at], x[at], w)
    R.assert_within(dw, ref, bound, "dw")  # (a zero row rounds nothing)
    del x, dy
    torch.cuda.empty_cache()


def test_products_on_two_streams_at_once(senmoe, torch):
    """Every tile form and the elementwise kernels queued on two streams side by
    side, other sizes on each: the bits of the same calls one after the other."""
    def calls(seed, rows, k, out, stream=None):
        s = [_normal(torch, seed + i, *shape, scale=sc) for i, (shape, sc) in enumerate(
            [((rows, k), 1), ((2 * out, k), k ** -0.5), ((rows, out), 0.5), ((rows, 2 * out), 1), ((4, out, k), k ** -0.5)])]
        off = torch.tensor([0, rows // 3, rows // 3, rows - 5, rows], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()

        def run(stream):
            got = []
            for path in (senmoe.LINEAR_AUTO, senmoe.LINEAR_TCGEN05_ONE, senmoe.LINEAR_TCGEN05_PAIR):
                got.append(senmoe.linear(s[0], s[1], activation="swiglu", path=path, stream=stream))
                got += senmoe.linear_backward(s[2], s[0], s[1], preact=s[3], activation="swiglu", bias=True, path=path,
                                              stream=stream)
                got.append(senmoe.grouped_linear(s[0], s[4], off, path=path, stream=stream))
                got += senmoe.grouped_linear_backward(s[2], s[0], s[4], off, bias=True, path=path, stream=stream)
            return got
        return run
    a, b = calls(1, 1300, 512, 320), calls(7, 210, 1024, 264)
    want = a(None), b(None)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        got = a(sa), b(sb)
    sa.synchronize()
    sb.synchronize()
    senmoe.linear_check()
    for w, g in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(w, g))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 31, 33, 511, 512, 513, 769, 16384, 16385, 40001])
@pytest.mark.parametrize("out,stride", [(136, 136), (33, 40), (257, 257)])
def test_bias_gradient_without_an_activation(senmoe, torch, rows, out, stride, dtype):
    """Where dW does not take the sums: not asked for, or on the copying kernels."""
    import linear_ref as R
    k = 24
    dy = _normal(torch, 1, rows, stride, dtype=dtype)[:, :out]
    x, w = _normal(torch, 2, rows, k, dtype=dtype), _normal(torch, 3, out, k, dtype=dtype)
    ref, size = dy.double().sum(0), dy.double().abs().sum(0)
    err = (rows + 8) * 2.0 ** -23 * size
    bound = err + R.HALF_UNIT[x.dtype] * (ref.abs() + err) + R.TINY[x.dtype]
    for path, dw in ((senmoe.LINEAR_AUTO, False), (senmoe.LINEAR_ANY, True), (senmoe.LINEAR_AUTO, True)):
        db = senmoe.linear_backward(dy, x, w, bias=True, need_dx=False, need_dweight=dw, path=path)[2]
        R.assert_within(db, ref, bound, "db")
