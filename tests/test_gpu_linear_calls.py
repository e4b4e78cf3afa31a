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
