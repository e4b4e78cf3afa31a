"""The 16-bit linear products and their gradients on the GPU, dense and
grouped, against float64 with elementwise bounds (linear_ref.py)."""
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


@pytest.fixture(params=["any", "auto"])
def path(request, senmoe):
    return {"any": senmoe.LINEAR_ANY, "auto": senmoe.LINEAR_AUTO}[request.param]


DTYPES = ["bfloat16", "float16"]


def _make(torch, rows, k, wide, dtype, seed=0, experts=None, std=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + k * 3 + wide)
    dt = getattr(torch, dtype)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)
    lead = () if experts is None else (experts,)
    return {"x": normal(rows, k), "w": normal(*lead, wide, k, scale=std / k ** 0.5), "b": normal(*lead, wide, scale=0.3),
            "r": normal(rows, wide), "dy": normal(rows, wide, scale=0.5), "z": normal(rows, wide)}


def _offsets(torch, counts, first=0):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def _wide(activation, out):
    return out * (2 if activation in ("swiglu", "geglu") else 1)


# sizes at which tiles, their halves and single elements end, and the next ones
DENSE = [(1, 1, 1), (1, 64, 128), (1, 2048, 64), (2, 8, 16), (3, 40, 24), (17, 129, 65), (63, 64, 64), (64, 65, 127),
         (65, 256, 200), (127, 72, 520), (128, 128, 128), (129, 136, 264), (257, 1000, 136), (300, 200, 1), (513, 64, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,out", DENSE)
def test_linear_sizes(senmoe, torch, path, rows, k, out, dtype):
    import linear_ref as R
    s = _make(torch, rows, k, out, dtype)
    y = senmoe.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], path=path)
    ref, bound, _, _ = R.forward(s["x"], s["w"], None, s["b"], s["r"])
    R.assert_within(y, ref, bound, "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu"])
@pytest.mark.parametrize("rows,k,out", [(1, 256, 136), (70, 192, 72), (200, 320, 264)])
def test_linear_activations(senmoe, torch, path, activation, rows, k, out, dtype):
    import linear_ref as R
    wide = _wide(activation, out)
    s = _make(torch, rows, k, wide, dtype, std=2.0)
    r = s["r"][:, :out].contiguous()
    y, z = senmoe.linear(s["x"], s["w"], bias=s["b"], residual=r, activation=activation, save_preact=True, path=path)
    ref, bound, zr, zb = R.forward(s["x"], s["w"], None, s["b"], r, activation)
    R.assert_within(z, zr, zb, "preact")
    R.assert_within(y, ref, bound, "y")
    plain = senmoe.linear(s["x"], s["w"], activation=activation, path=path)
    ref, bound, _, _ = R.forward(s["x"], s["w"], None, None, None, activation)
    R.assert_within(plain, ref, bound, "y without bias and residual")


GROUPS = [
    [5], [0, 0, 7], [1, 1, 1, 1], [0, 3, 0, 130, 1, 0, 64, 65], [63, 64, 65, 127, 128, 129],
    [255, 0, 256, 257, 16, 15, 17], [0] * 40 + [300] + [0] * 23, [600, 1, 0, 2], [0, 0, 0],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: f"{len(c)}g{sum(c)}r")
@pytest.mark.parametrize("k,out,activation", [(72, 136, "none"), (256, 64, "swiglu"), (130, 33, "geglu")])
def test_grouped_linear(senmoe, torch, path, counts, k, out, activation, dtype):
    import linear_ref as R
    rows, wide = sum(counts), _wide(activation, out)
    s = _make(torch, rows, k, wide, dtype, experts=len(counts))
    off = _offsets(torch, counts)
    y, z = senmoe.grouped_linear(s["x"], s["w"], off, bias=s["b"], activation=activation, save_preact=True, path=path)
    ref, bound, zr, zb = R.forward(s["x"], s["w"], off.tolist(), s["b"], None, activation)
    R.assert_within(z, zr, zb, "preact")
    R.assert_within(y, ref, bound, "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: f"{len(c)}g{sum(c)}r")
@pytest.mark.parametrize("k,out,activation", [(72, 136, "none"), (256, 64, "swiglu"), (130, 33, "geglu")])
def test_grouped_backward(senmoe, torch, path, counts, k, out, activation, dtype):
    import linear_ref as R
    rows, wide = sum(counts), _wide(activation, out)
    s = _make(torch, rows, k, wide, dtype, experts=len(counts))
    off, dy = _offsets(torch, counts), s["dy"][:, :out].contiguous()
    z = None if activation == "none" else s["z"]
    dx, dw, db = senmoe.grouped_linear_backward(dy, s["x"], s["w"], off, preact=z, activation=activation, bias=True,
                                                path=path)
    for got, (ref, bound), what in zip((dx, dw, db), R.backward(dy, s["x"], s["w"], off.tolist(), z, activation),
                                       ("dx", "dw", "db")):
        R.assert_within(got, ref, bound, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu"])
@pytest.mark.parametrize("rows,k,out", [(1, 64, 40), (67, 136, 72), (600, 200, 264), (33, 129, 65)])
def test_linear_backward(senmoe, torch, path, activation, rows, k, out, dtype):
    import linear_ref as R
    wide = _wide(activation, out)
    s = _make(torch, rows, k, wide, dtype)
    dy, z = s["dy"][:, :out].contiguous(), None if activation == "none" else s["z"]
    got = senmoe.linear_backward(dy, s["x"], s["w"], preact=z, activation=activation, bias=True, path=path)
    for v, (ref, bound), what in zip(got, R.backward(dy, s["x"], s["w"], None, z, activation), ("dx", "dw", "db")):
        R.assert_within(v, ref, bound, what)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "swiglu", "geglu"])
def test_gradients_against_differences(senmoe, torch, activation):
    """<grad, v> against (L(p + h v) - L(p - h v)) / 2h of the float64
    product's loss L = sum dy * y.  The difference's own error is O(h^2) =
    1e-8 of terms of order 1; the kernel's is that of the elementwise bounds,
    summed over the direction."""
    import linear_ref as R
    counts, k, out = [40, 0, 33, 1], 64, 48
    rows, wide = sum(counts), _wide(activation, out)
    s = _make(torch, rows, k, wide, "float16", experts=len(counts))
    off, dy = _offsets(torch, counts), s["dy"][:, :out].contiguous()
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    z64 = torch.cat([x[a:c] @ w[e].t() + b[e] for e, a, c in R.groups(off.tolist(), rows)])
    # the loss at the preact that the kernel is given: z rounded to fp16, b moved to match
    z16 = z64.half()
    got = senmoe.grouped_linear_backward(dy, s["x"], s["w"], off, preact=z16, activation=activation, bias=True)
    shift = z16.double() - z64

    def loss_at(x, w, b):
        z = torch.cat([x[a:c] @ w[e].t() + b[e] for e, a, c in R.groups(off.tolist(), rows)]) + shift
        return (R.act(activation, z) * dy.double()).sum()
    bounds = [bound for _, bound in R.backward(dy, s["x"], s["w"], off.tolist(), z16, activation)]
    g = torch.Generator(device="cuda").manual_seed(5)
    h = 1e-4
    for i in range(3):
        p = [x, w, b]
        v = torch.randn(p[i].shape, generator=g, device="cuda", dtype=torch.float64)
        hi, lo = list(p), list(p)
        hi[i], lo[i] = p[i] + h * v, p[i] - h * v
        diff = (loss_at(*hi) - loss_at(*lo)) / (2 * h)
        mine = (got[i].double() * v).sum()
        allow = (bounds[i] * v.abs()).sum() + 1e-5 * v.norm() ** 2
        assert abs(float(mine - diff)) <= float(allow)


def test_rows_outside_the_groups_are_zero(senmoe, torch, path):
    """A rank's slice of the offsets: earlier and later rows belong to others."""
    import linear_ref as R
    counts, first, rows, k, out = [30, 0, 45], 21, 140, 128, 72
    s = _make(torch, rows, k, 2 * out, "bfloat16", experts=3)
    off = _offsets(torch, counts, first)
    s["x"][:first] = float("nan")
    s["x"][first + 75:] = float("inf")
    y, z = senmoe.grouped_linear(s["x"], s["w"], off, activation="swiglu", save_preact=True, path=path)
    dy = s["dy"][:, :out].contiguous()
    dy[:first] = float("nan")
    dx, dw, db = senmoe.grouped_linear_backward(dy, s["x"], s["w"], off, preact=s["z"], activation="swiglu", bias=True,
                                                path=path)
    for v in (y, z, dx):
        assert (v[:first] == 0).all() and (v[first + 75:] == 0).all()
    inner = slice(first, first + 75)
    loc = [o - first for o in off.tolist()]
    ref, bound, _, _ = R.forward(s["x"][inner], s["w"], loc, None, None, "swiglu")
    R.assert_within(y[inner], ref, bound, "y")
    back = R.backward(dy[inner], s["x"][inner], s["w"], loc, s["z"][inner], "swiglu")
    for got, (r, bd), what in zip((dx[inner], dw, db), back, ("dx", "dw", "db")):
        R.assert_within(got, r, bd, what)


def test_nonfinite_rows_stay_in_their_group(senmoe, torch, path):
    import linear_ref as R
    counts, k, out = [37, 5, 61], 96, 80
    rows = sum(counts)
    s = _make(torch, rows, k, out, "bfloat16", experts=3)
    off = _offsets(torch, counts)
    x, dy = s["x"].clone(), s["dy"].clone()
    x[38], dy[39] = float("nan"), float("inf")  # group 1
    keep = torch.tensor([i for i in range(rows) if not 37 <= i < 42], device="cuda")
    y = senmoe.grouped_linear(x, s["w"], off, path=path)
    dx, dw, db = senmoe.grouped_linear_backward(dy, x, s["w"], off, bias=True, path=path)
    ref, bound, _, _ = R.forward(s["x"], s["w"], off.tolist())
    R.assert_within(y[keep], ref[keep], bound[keep], "y")
    assert torch.isnan(y[38]).all() and torch.isfinite(y[37]).all()
    (rx, bx), (rw, bw), (rb, bb) = R.backward(s["dy"], s["x"], s["w"], off.tolist())
    R.assert_within(dx[keep], rx[keep], bx[keep], "dx")
    for e in (0, 2):
        R.assert_within(dw[e], rw[e], bw[e], "dw")
        R.assert_within(db[e], rb[e], bb[e], "db")
    assert not torch.isfinite(dw[1]).any() and not torch.isfinite(db[1]).any()


def test_bad_offsets_touch_nothing_outside(senmoe, torch, path):
    """Offsets below 0, past the rows and falling are clamped; the call ends
    and later calls are right."""
    import linear_ref as R
    rows, k, out = 100, 64, 64
    s = _make(torch, rows, k, out, "bfloat16", experts=4)
    for bad in ([-5, 20, 30, 40, 100], [0, 20, 30, 40, 2 ** 31 - 1], [0, 90, 10, 50, 20], [100, 0, 0, 0, 0]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        senmoe.grouped_linear(s["x"], s["w"], off, path=path)
        senmoe.grouped_linear_backward(s["dy"], s["x"], s["w"], off, bias=True, path=path)
    senmoe.linear_check()
    off = _offsets(torch, [25, 25, 25, 25])
    ref, bound, _, _ = R.forward(s["x"], s["w"], off.tolist())
    R.assert_within(senmoe.grouped_linear(s["x"], s["w"], off, path=path), ref, bound, "y")


@pytest.mark.parametrize("shift", [0, 1, 4, 8])
def test_strided_and_unaligned_operands(senmoe, torch, path, shift):
    """Columns `shift` on of wider tensors: row strides and bases off the
    16-byte grid, outputs written in place into a wider tensor."""
    import linear_ref as R
    rows, k, out = 70, 96, 88
    big = _make(torch, rows, k + 24, out + 16, "bfloat16", experts=3)
    x, w = big["x"][:, shift:shift + k], big["w"][:, 5:5 + out, shift:shift + k]
    off = _offsets(torch, [30, 9, 31])
    buf = torch.full((rows, out + 32), 7.0, dtype=torch.bfloat16, device="cuda")
    y = senmoe.grouped_linear(x, w, off, out=buf[:, shift:shift + out], path=path)
    ref, bound, _, _ = R.forward(x, w, off.tolist())
    R.assert_within(y, ref, bound, "y")
    assert (buf[:, :shift] == 7).all() and (buf[:, shift + out:] == 7).all()
    dy, z = big["dy"][:, shift:shift + out], big["z"][:, shift:shift + out]
    got = senmoe.grouped_linear_backward(dy, x, w, off, preact=z, activation="gelu", bias=True, path=path)
    for v, (r, b), what in zip(got, R.backward(dy, x, w, off.tolist(), z, "gelu"), ("dx", "dw", "db")):
        R.assert_within(v, r, b, what)


def test_other_layouts_and_leading_dimensions(senmoe, torch):
    import linear_ref as R
    s = _make(torch, 6 * 5, 64, 40, "bfloat16")
    w = s["w"].t().contiguous().t()  # columns of W contiguous
    x = s["x"].reshape(6, 5, 64)
    y = senmoe.linear(x, w, bias=s["b"])
    assert y.shape == (6, 5, 40)
    ref, bound, _, _ = R.forward(s["x"], s["w"], None, s["b"])
    R.assert_within(y.reshape(30, 40), ref, bound, "y")
    one = senmoe.linear(s["x"][0], s["w"], bias=s["b"])
    assert one.shape == (40,)
    R.assert_within(one, ref[0], bound[0], "one row")
    same = s["x"][:1].expand(30, 64)  # a broadcast row
    y = senmoe.linear(same, s["w"], bias=s["b"])
    R.assert_within(y, ref[:1].expand(30, 40), bound[:1].expand(30, 40), "broadcast x")
    dx, dw, db = senmoe.linear_backward(s["dy"].reshape(6, 5, 40).transpose(0, 1).contiguous().transpose(0, 1), x, w,
                                        bias=True)
    assert dx.shape == x.shape
    (rx, bx), (rw, bw), _ = R.backward(s["dy"], s["x"], s["w"])
    R.assert_within(dx.reshape(30, 64), rx, bx, "dx")
    R.assert_within(dw, rw, bw, "dw")


def test_row_offsets_past_32_bits(senmoe, torch, path):
    """Rows 2^15 elements apart, so the last ones lie past element 2^31."""
    import linear_ref as R
    rows, k, out, stride = 66000, 64, 16, 32768
    base = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((rows, k), (stride, 1))
    s = _make(torch, rows, k, out, "bfloat16")
    x.copy_(s["x"])
    off = _offsets(torch, [65000, 0, 1000])
    w = _make(torch, 1, k, out, "bfloat16", experts=3)["w"]
    y = senmoe.grouped_linear(x, w, off, path=path)
    ref, bound, _, _ = R.forward(s["x"], w, off.tolist())
    R.assert_within(y, ref, bound, "y")
    dx, dw, _ = senmoe.grouped_linear_backward(s["dy"], x, w, off, path=path)
    (rx, bx), (rw, bw), _ = R.backward(s["dy"], s["x"], w, off.tolist())
    R.assert_within(dx, rx, bx, "dx")
    R.assert_within(dw, rw, bw, "dw")


def test_no_rows(senmoe, torch, path):
    s = _make(torch, 0, 64, 48, "bfloat16", experts=2)
    off = _offsets(torch, [0, 0])
    assert senmoe.grouped_linear(s["x"], s["w"], off, path=path).shape == (0, 48)
    dx, dw, db = senmoe.grouped_linear_backward(s["dy"], s["x"], s["w"], off, bias=True, path=path)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    dx, dw, db = senmoe.linear_backward(s["dy"], s["x"], s["w"][0], bias=True, path=path)
    assert (dw == 0).all() and (db == 0).all()


def test_parts_of_the_gradient(senmoe, torch):
    s = _make(torch, 90, 64, 48, "bfloat16")
    dx, dw, db = senmoe.linear_backward(s["dy"], s["x"], s["w"], bias=True)
    only = senmoe.linear_backward(s["dy"], s["x"], s["w"], need_dweight=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None
    only = senmoe.linear_backward(s["dy"], s["x"], s["w"], need_dx=False)
    assert only[0] is None and torch.equal(only[1], dw)


def test_many_groups(senmoe, torch, path):
    import linear_ref as R
    E, k, out = 1024, 64, 24
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 6, (E,), generator=g).tolist()
    counts[1023] = 70
    rows = sum(counts)
    s = _make(torch, rows, k, out, "bfloat16", experts=E)
    off = _offsets(torch, counts)
    y = senmoe.grouped_linear(s["x"], s["w"], off, bias=s["b"], path=path)
    ref, bound, _, _ = R.forward(s["x"], s["w"], off.tolist(), s["b"])
    R.assert_within(y, ref, bound, "y")
    got = senmoe.grouped_linear_backward(s["dy"], s["x"], s["w"], off, bias=True, path=path)
    for v, (r, b), what in zip(got, R.backward(s["dy"], s["x"], s["w"], off.tolist()), ("dx", "dw", "db")):
        R.assert_within(v, r, b, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,out,activation", [(1, 2048, 2048, "none"), (8, 2048, 1536, "swiglu"),
                                                  (40, 2056, 1032, "gelu"), (1031, 704, 2816, "geglu"),
                                                  (2500, 520, 1160, "silu")])
def test_linear_model_sizes(senmoe, torch, rows, k, out, activation, dtype):
    import linear_ref as R
    s = _make(torch, rows, k, _wide(activation, out), dtype)
    r = s["r"][:, :out]
    y, z = senmoe.linear(s["x"], s["w"], bias=s["b"], residual=r, activation=activation, save_preact=True)
    ref, bound, zr, zb = R.forward(s["x"], s["w"], None, s["b"], r, activation)
    R.assert_within(z, zr, zb, "preact")
    R.assert_within(y, ref, bound, "y")
    dy, z = s["dy"][:, :out], None if activation == "none" else s["z"]
    got = senmoe.linear_backward(dy, s["x"], s["w"], preact=z, activation=activation, bias=True)
    for v, (r, b), what in zip(got, R.backward(dy, s["x"], s["w"], None, z, activation), ("dx", "dw", "db")):
        R.assert_within(v, r, b, what)


@pytest.mark.parametrize("tokens,experts,top_k,k,out,activation", [(1, 128, 8, 2048, 768, "swiglu"),
                                                                   (64, 128, 8, 768, 1024, "none"),
                                                                   (700, 16, 4, 1024, 264, "geglu"),
                                                                   (3000, 8, 2, 264, 520, "relu")])
def test_grouped_over_dispatched_tokens(senmoe, torch, tokens, experts, top_k, k, out, activation):
    """router -> dispatch -> grouped product of the gathered rows, as the block chains them."""
    import linear_ref as R
    s = _make(torch, tokens, k, _wide(activation, out), "bfloat16", experts=experts)
    rw = _make(torch, 1, k, experts, "bfloat16", seed=9)["w"]
    ids, _ = senmoe.router(s["x"], rw, top_k)
    perm, _, off, _ = senmoe.dispatch(ids, experts)
    xs = s["x"][(perm // top_k).long()]
    y = senmoe.grouped_linear(xs, s["w"], off, activation=activation)
    ref, bound, _, _ = R.forward(xs, s["w"], off.tolist(), None, None, activation)
    R.assert_within(y, ref, bound, "y")
    dy = _make(torch, xs.shape[0], 8, out, "bfloat16")["dy"]
    z = None if activation == "none" else _make(torch, xs.shape[0], 8, _wide(activation, out), "bfloat16")["z"]
    dx, dw, _ = senmoe.grouped_linear_backward(dy, xs, s["w"], off, preact=z, activation=activation)
    (rx, bx), (rw_, bw), _ = R.backward(dy, xs, s["w"], off.tolist(), z, activation)
    R.assert_within(dx, rx, bx, "dx")
    R.assert_within(dw, rw_, bw, "dw")


@pytest.mark.parametrize("rows,k,out", [(1, 2048, 512), (100, 512, 256), (900, 256, 512)])
def test_repeat_other_stream_and_graph_agree(senmoe, torch, rows, k, out):
    """The same bits again, on a stream of its own, and from a captured graph."""
    s = _make(torch, rows, k, out, "bfloat16")

    def both(stream=None):
        y, z = senmoe.linear(s["x"], s["w"], bias=s["b"], activation="silu", save_preact=True, stream=stream)
        return (y, z, *senmoe.linear_backward(s["dy"], s["x"], s["w"], preact=s["z"], activation="silu", bias=True,
                                              stream=stream))
    first = both()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = both(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for t in held:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, held))
    senmoe.linear_check()


def test_python_refusals(senmoe, torch):
    s = _make(torch, 8, 64, 32, "bfloat16", experts=2)
    off = _offsets(torch, [4, 4])
    E = senmoe.SenMoeError
    with pytest.raises(E):
        senmoe.grouped_linear(s["x"][:, :32], s["w"], off)
    with pytest.raises(TypeError):
        senmoe.grouped_linear(s["x"], s["w"].half(), off)
    with pytest.raises(E, match="even"):
        senmoe.linear(s["x"], s["w"][0, :31], activation="swiglu")
    with pytest.raises(E, match="bias"):
        senmoe.grouped_linear(s["x"], s["w"], off, bias=s["b"][0])
    with pytest.raises(E, match="residual"):
        senmoe.linear(s["x"], s["w"][0], residual=s["r"][:4])
    with pytest.raises(E, match="out"):
        senmoe.linear(s["x"], s["w"][0], out=torch.empty(32, 8, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(E, match="preact"):
        senmoe.linear_backward(s["dy"], s["x"], s["w"][0], activation="gelu")
    with pytest.raises(E):
        senmoe.linear_backward(s["dy"][:4], s["x"], s["w"][0])


# Every kernel and tile form on shapes that each can take: rows and features
# that end inside tiles, chunks and 64-element boxes, K shorter than a block
# and not a multiple of one.
FORM_SHAPES = [(1, 64, 128), (5, 8, 16), (16, 520, 136), (33, 72, 40), (64, 256, 264), (70, 264, 200), (161, 1032, 520),
               (300, 192, 328)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["TCGEN05", "SMALL", "TCGEN05_ONE", "TCGEN05_PAIR", "TCGEN05_SPLIT"])
@pytest.mark.parametrize("activation", ["none", "swiglu"])
@pytest.mark.parametrize("rows,k,out", FORM_SHAPES)
def test_every_form(senmoe, torch, form, rows, k, out, activation, dtype):
    import linear_ref as R
    form, wide = getattr(senmoe, "LINEAR_" + form), _wide(activation, out)
    s = _make(torch, rows, k, wide, dtype)
    r = s["r"][:, :out].contiguous()
    y, z = senmoe.linear(s["x"], s["w"], bias=s["b"], residual=r, activation=activation, save_preact=True, path=form)
    ref, bound, zr, zb = R.forward(s["x"], s["w"], None, s["b"], r, activation)
    R.assert_within(z, zr, zb, "preact")
    R.assert_within(y, ref, bound, "y")
    dy, z = s["dy"][:, :out].contiguous(), None if activation == "none" else s["z"]
    got = senmoe.linear_backward(dy, s["x"], s["w"], preact=z, activation=activation, bias=True, path=form)
    for v, (ref, bound), what in zip(got, R.backward(dy, s["x"], s["w"], None, z, activation), ("dx", "dw", "db")):
        R.assert_within(v, ref, bound, what)
    senmoe.linear_check()


@pytest.mark.parametrize("form", ["TCGEN05", "SMALL", "TCGEN05_ONE", "TCGEN05_PAIR"])
@pytest.mark.parametrize("activation", ["none", "geglu"])
@pytest.mark.parametrize("counts", GROUPS[:8], ids=lambda c: f"{len(c)}g{sum(c)}r")
@pytest.mark.parametrize("k,out", [(72, 136), (256, 328)])
def test_every_form_grouped(senmoe, torch, form, counts, k, out, activation):
    import linear_ref as R
    form, wide, rows = getattr(senmoe, "LINEAR_" + form), _wide(activation, out), sum(counts)
    s = _make(torch, rows + 9, k, wide, "bfloat16", experts=len(counts))
    off = _offsets(torch, counts, 4)  # rows 0-3 and the last 5 in no group
    y = senmoe.grouped_linear(s["x"], s["w"], off, bias=s["b"], activation=activation, path=form)
    ref, bound, _, _ = R.forward(s["x"], s["w"], off.tolist(), s["b"], None, activation)
    assert (y[:4] == 0).all() and (y[4 + rows:] == 0).all()
    R.assert_within(y[4:4 + rows], ref[4:4 + rows], bound[4:4 + rows], "y")
    dy, z = s["dy"][:, :out].contiguous(), None if activation == "none" else s["z"]
    got = senmoe.grouped_linear_backward(dy, s["x"], s["w"], off, preact=z, activation=activation, bias=True, path=form)
    assert (got[0][:4] == 0).all() and (got[0][4 + rows:] == 0).all()
    for v, (ref, bound), what in zip(got, R.backward(dy, s["x"], s["w"], off.tolist(), z, activation),
                                     ("dx", "dw", "db")):
        R.assert_within(v, ref, bound, what)
    senmoe.linear_check()


def test_k_split_over_a_group_that_is_empty_here(senmoe, torch):
    """A K split's cluster whose tile has fewer K blocks than CTAs, and
    clusters left without a tile by the groups' real counts."""
    import linear_ref as R
    s = _make(torch, 20, 72, 128, "bfloat16", experts=5)
    off = _offsets(torch, [0, 19, 0, 1, 0])
    y = senmoe.grouped_linear(s["x"], s["w"], off, bias=s["b"], path=senmoe.LINEAR_TCGEN05_SPLIT)
    ref, bound, _, _ = R.forward(s["x"], s["w"], off.tolist(), s["b"])
    R.assert_within(y, ref, bound, "y")
    dx, dw, db = senmoe.grouped_linear_backward(s["dy"], s["x"], s["w"], off, bias=True,
                                                path=senmoe.LINEAR_TCGEN05_SPLIT)
    for v, (ref, bound), what in zip((dx, dw, db), R.backward(s["dy"], s["x"], s["w"], off.tolist()),
                                     ("dx", "dw", "db")):
        R.assert_within(v, ref, bound, what)


def test_unsupported_forms(senmoe, torch):
    s = _make(torch, 40, 33, 24, "bfloat16")
    for form in (senmoe.LINEAR_TCGEN05, senmoe.LINEAR_TCGEN05_PAIR, senmoe.LINEAR_SMALL):
        with pytest.raises(senmoe.SenMoeError) as e:
            senmoe.linear(s["x"], s["w"], path=form)
        assert e.value.status == senmoe.ERR_UNSUPPORTED
    s = _make(torch, 4000, 64, 4096, "bfloat16")
    with pytest.raises(senmoe.SenMoeError) as e:
        senmoe.linear(s["x"], s["w"], path=senmoe.LINEAR_TCGEN05_SPLIT)
    assert e.value.status == senmoe.ERR_UNSUPPORTED


@pytest.mark.parametrize("activation", ["none", "geglu"])
@pytest.mark.parametrize("rows", [257, 263, 320, 1031, 1088])
def test_rows_past_whole_tiles(senmoe, torch, rows, activation):
    """A few rows past a multiple of the widest tile, which may go to another
    kernel; before and after other work on the stream."""
    import linear_ref as R
    k, out = 512, 2112
    wide = _wide(activation, out)
    s = _make(torch, rows, k, wide, "bfloat16")
    r = s["r"][:, :out].contiguous()
    ref, bound, zr, zb = R.forward(s["x"], s["w"], None, s["b"], r, activation)
    for _ in range(3):
        x = s["x"] + 0  # written just before the call, read and overwritten right after
        y, z = senmoe.linear(x, s["w"], bias=s["b"], residual=r, activation=activation, save_preact=True)
        x.zero_()
        copy = y + 0
        R.assert_within(z, zr, zb, "preact")
        R.assert_within(copy, ref, bound, "y")


def test_a_long_chain_of_calls(senmoe, torch):
    """A thousand calls of several kernels each, queued without waiting: the
    last one's results are the first one's."""
    s = _make(torch, 1500, 512, 1088, "bfloat16")
    t = _make(torch, 40, 1024, 512, "bfloat16")

    def calls():
        y, z = senmoe.linear(s["x"], s["w"], bias=s["b"], activation="gelu", save_preact=True)
        g = senmoe.linear_backward(s["dy"], s["x"], s["w"], preact=s["z"], activation="gelu", bias=True)
        return (y, z, *g, senmoe.linear(t["x"], t["w"]), *senmoe.linear_backward(t["dy"], t["x"], t["w"])[:2])
    first = calls()
    for _ in range(1000):
        last = calls()
    senmoe.linear_check()
    assert all(torch.equal(a, b) for a, b in zip(first, last))
